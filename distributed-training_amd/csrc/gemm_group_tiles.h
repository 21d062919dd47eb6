// The kernels behind gemm_group.h.
#pragma once

#include "gemm_direct_tile.h"
#include "gemm_group.h"
#include "gemm_rows.h"
#include "gemm_tiles.h"
#include "seqmath.h"

namespace dtmi {

// Blocks are dealt to the 8 XCDs in turn: this order gives each a contiguous range of
// tiles, whose operands its L2 then holds. The last tiles % 8 keep their place.
__device__ __forceinline__ int xcd_tile(int b, int tiles) {
  const int per = tiles >> 3;
  return b < 8 * per ? (b & 7) * per + (b >> 3) : b;
}

// The tile of the launch's unit v of those past the split ones.
__device__ __forceinline__ int whole_tile(const GroupArgs& a, int v) {
  const int work = a.work - a.cut;
  return a.cut + (a.equal && v < work ? xcd_tile(v, work) : v);
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

// The task of the launch's tile v and the tile's place in that task's grid. Every lane
// holds the first tile of one task.
__device__ __forceinline__ void group_tile(const GroupArgs& a, int bm, int v, int& task, int& tm, int& tn) {
  const int lane = threadIdx.x & 63;
  const int first = lane < a.count ? a.first[lane] : 0x7fffffff;
  task = __builtin_amdgcn_readfirstlane(63 - __builtin_clzll(__ballot(first <= v)));
  group_coords(v - a.first[task], (a.t[task].M + bm - 1) / bm, (a.t[task].N + bm - 1) / bm, a.sym, tm, tn);
}

__device__ __forceinline__ int pad_up(int n, int pad) { return (n + pad - 1) / pad * pad; }

// One output element: s (alpha v + beta D) + gamma C.
template <typename T>
struct GroupEpi {
  T alpha, beta, gamma, s;
  int dmode;
  bool mirror, turned;
  const T* D;
  T* C;
  int64_t ldd, ldc;
  int M, N;  // what is stored
  __device__ __forceinline__ T value(T v, T d, T old) const {
    v = alpha * v;
    if (dmode == kDMatrix) v = fma(beta, d, v);
    if (dmode == kDRow) v = v + d;
    v = s * v;
    if (gamma != T(0)) v = fma(gamma, old, v);
    return v;
  }
  __device__ __forceinline__ T* place(int64_t m, int64_t n) const { return C + (turned ? n * ldc + m : m * ldc + n); }
  __device__ __forceinline__ T at(int64_t m, int64_t n, T v) const {
    const T d = dmode == kDMatrix ? D[m * ldd + n] : dmode == kDRow ? D[n] : T(0);
    return value(v, d, gamma != T(0) ? *place(m, n) : T(0));
  }
  __device__ __forceinline__ void store(int64_t m, int64_t n, T v) const {
    v = at(m, n, v);
    *place(m, n) = v;
    if (mirror) *place(n, m) = v;
  }
};

template <typename T>
__device__ __forceinline__ GroupEpi<T> group_epi(const GroupArgs& a, const GroupTask& k, bool mirror) {
  const bool zeros = a.padc == a.pad;
  return {(T)a.alpha, (T)a.beta, (T)a.gamma, (T)k.s,
          k.D ? a.dmode : (int)kDNone, mirror, k.turned != 0, (const T*)k.D, (T*)k.C,
          (int64_t)pad_up(k.N, a.pad), (int64_t)pad_up(k.turned ? k.M : k.N, a.padc),
          zeros ? pad_up(k.M, a.pad) : k.M, zeros ? pad_up(k.N, a.pad) : k.N};
}

// A column sum, added to the old one where C is.
template <typename T>
__device__ __forceinline__ void put_colsum(const GroupArgs& a, const GroupTask& k, int64_t n, T v) {
  T* d = (T*)k.D + n;
  *d = a.gamma != 0.0 ? fma((T)a.gamma, *d, v) : v;
}

// A wave tile's accumulators through the epilogue.
template <typename T, int TW>
__device__ __forceinline__ void group_write(const GroupEpi<T>& e, const typename MF<T>::acc_t (&acc)[TW][TW],
                                            int64_t wm, int64_t wn, int g, int c) {
  using MFT = MF<T>;
  constexpr int MT = MFT::MT, NACC = MFT::NACC, W = TW * MT;
  if constexpr (sizeof(T) == 4) {
    if (wm + W <= e.M && wn + W <= e.N) {
      // a wave tile in range: buffer accesses off its corner, one lane offset and a
      // wave-uniform offset per element (as write_acc); D and C of a row of MFMA tiles
      // are read before its first store. The transposed image, where there is one: a
      // lane's registers 4q .. 4q + 3 are four rows of one column, so four elements in a
      // row of it, 16 bytes where its rows allow.
      const Rsrc rc = make_rsrc(e.turned ? e.C : e.C + wm * e.ldc + wn, ~0ull);
      const Rsrc rd = make_rsrc(e.dmode == kDMatrix ? e.D + wm * e.ldd + wn : e.C, ~0ull);
      const uint32_t voff = (uint32_t)((4 * g * e.ldc + c) * 4), doff = (uint32_t)((4 * g * e.ldd + c) * 4);
      const bool wide = e.ldc % 4 == 0 && aligned(e.C, 16);
      float row[TW];
#pragma unroll
      for (int j = 0; j < TW; ++j) row[j] = e.dmode == kDRow ? e.D[wn + j * MT + c] : 0.f;
#pragma unroll
      for (int i = 0; i < TW; ++i) {
        float d[TW][NACC], old[TW][NACC];
        float* image[TW];
#pragma unroll
        for (int j = 0; j < TW; ++j) {
          image[j] = e.C + (wn + j * MT + c) * e.ldc + wm + i * MT + 4 * g;
#pragma unroll
          for (int r = 0; r < NACC; ++r) {
            d[j][r] = row[j];
            old[j][r] = 0.f;
          }
        }
        if (e.dmode == kDMatrix)
#pragma unroll
          for (int j = 0; j < TW; ++j)
#pragma unroll
            for (int r = 0; r < NACC; ++r)
              d[j][r] = buf_load1(rd, doff, (uint32_t)(((i * MT + MFT::row(r, 0)) * e.ldd + j * MT) * 4));
        if (e.gamma != 0.f) {
          if (e.turned) {
#pragma unroll
            for (int j = 0; j < TW; ++j)
#pragma unroll
              for (int r = 0; r < NACC; ++r) old[j][r] = image[j][8 * (r / 4) + r % 4];
          } else {
#pragma unroll
            for (int j = 0; j < TW; ++j)
#pragma unroll
              for (int r = 0; r < NACC; ++r)
                old[j][r] = buf_load1(rc, voff, (uint32_t)(((i * MT + MFT::row(r, 0)) * e.ldc + j * MT) * 4));
          }
        }
#pragma unroll
        for (int j = 0; j < TW; ++j) {
          float v[NACC];
#pragma unroll
          for (int r = 0; r < NACC; ++r) v[r] = e.value(acc[i][j][r], d[j][r], old[j][r]);
          if (!e.turned)
#pragma unroll
            for (int r = 0; r < NACC; ++r)
              buf_store1(v[r], rc, voff, (uint32_t)(((i * MT + MFT::row(r, 0)) * e.ldc + j * MT) * 4));
          if (e.turned || e.mirror) {
            if (wide) {
#pragma unroll
              for (int q = 0; q < NACC / 4; ++q)
                *reinterpret_cast<f32x4*>(image[j] + 8 * q) = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            } else {
#pragma unroll
              for (int r = 0; r < NACC; ++r) image[j][8 * (r / 4) + r % 4] = v[r];
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
      if (n >= e.N) continue;
#pragma unroll
      for (int r = 0; r < NACC; ++r) {
        const int64_t m = wm + i * MT + MFT::row(r, g);
        if (m < e.M) e.store(m, n, acc[i][j][r]);
      }
    }
}

template <typename T, int BM, bool AKC, bool BKC, bool VEC>
__global__ void __launch_bounds__(256, 2) gemm_group_kernel(GroupArgs a) {
  using MFT = MF<T>;
  constexpr int MT = MFT::MT, NACC = MFT::NACC, BK = 64 / (int)sizeof(T);
  constexpr int W = BM / 2, TW = W / MT;
  extern __shared__ __attribute__((aligned(1024))) char lds_raw[];
  T* lds = reinterpret_cast<T*>(lds_raw);

  const int parts = a.cut * a.splits;
  int b = (int)blockIdx.x;
  if (b >= a.turn && b < a.turned) b = a.turn + a.turned - 1 - b;
  const bool cut = b >= a.before && b < a.before + parts;
  int split = 0, v;
  if (cut) {
    v = a.equal ? xcd_tile(b - a.before, parts) : b - a.before;
    split = v / a.cut;
    v -= split * a.cut;
  } else {
    v = whole_tile(a, b < a.before ? b : b - parts);
  }
  int ti, tm, tn;
  group_tile(a, BM, v, ti, tm, tn);
  const GroupTask k = a.t[ti];
  const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BM;
  const int Mp = pad_up(k.M, a.pad), Np = pad_up(k.N, a.pad), Kp = pad_up(k.K, a.pad);
  const int64_t kps = cut ? ((Kp + a.splits - 1) / a.splits + BK - 1) / BK * BK : Kp;
  const int64_t kbeg = split * kps < Kp ? split * kps : Kp;
  const int64_t kend = kbeg + kps < Kp ? kbeg + kps : Kp;

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane / MT, c = lane % MT;
  typename MFT::acc_t acc[TW][TW];
#pragma unroll
  for (int i = 0; i < TW; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j) acc[i][j] = typename MFT::acc_t(0);
  const bool take_colsum = a.dmode == kDColsum && tm == 0 && (int)threadIdx.x < BM;
  double csum = 0.0;
  dma_product<T, BM, BM, AKC, BKC, VEC, VEC>(acc, lds, (const T*)k.A, AKC ? Kp : Mp, Mp, m0, (const T*)k.B,
                                             BKC ? Kp : Np, Np, n0, kbeg, kend, sizeof(T) == 4 ? 2 : 4, take_colsum,
                                             csum);
  const int wm = (wave >> 1) * W, wn = (wave & 1) * W;
  if (cut) {  // the raw partial, tile by tile
    const int64_t slot = (int64_t)split * a.cut + v;
    T* P = (T*)a.ws + slot * (BM * BM);
#pragma unroll
    for (int i = 0; i < TW; ++i)
#pragma unroll
      for (int j = 0; j < TW; ++j)
#pragma unroll
        for (int r = 0; r < NACC; ++r) P[(wm + i * MT + MFT::row(r, g)) * BM + wn + j * MT + c] = acc[i][j][r];
    if (take_colsum) ((T*)a.csws)[slot * BM + threadIdx.x] = (T)csum;
    return;
  }
  if (take_colsum && k.D && n0 + threadIdx.x < k.N) put_colsum(a, k, n0 + threadIdx.x, (T)csum);
  group_write<T, TW>(group_epi<T>(a, k, a.sym && tm != tn), acc, m0 + wm, n0 + wn, g, c);
}

// The partials of a split tile, added in split order, and the epilogue: block (v, y)
// takes ROWS rows of tile v. Mirrored values go through LDS, so that both images
// are written along their rows.
template <typename T, int BM>
__global__ void __launch_bounds__(256) group_sum_kernel(GroupArgs a) {
  constexpr int PER = 8, ROWS = 256 * PER / BM;
  __shared__ T turned[ROWS][BM + 1];
  int ti, tm, tn;
  group_tile(a, BM, (int)blockIdx.x, ti, tm, tn);
  const GroupTask k = a.t[ti];
  const GroupEpi<T> e = group_epi<T>(a, k, false);
  const bool mirror = a.sym && tm != tn;
  const T* P = (const T*)a.ws + (int64_t)blockIdx.x * (BM * BM) + (int)blockIdx.y * (ROWS * BM) + threadIdx.x;
  const int64_t step = (int64_t)a.cut * (BM * BM);
  T v[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) v[u] = P[256 * u];
  int s = 1;
  for (; s + 1 < a.splits; s += 2) {
    T x[PER], y[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) x[u] = P[s * step + 256 * u];
#pragma unroll
    for (int u = 0; u < PER; ++u) y[u] = P[(s + 1) * step + 256 * u];
#pragma unroll
    for (int u = 0; u < PER; ++u) v[u] = (v[u] + x[u]) + y[u];
  }
  if (s < a.splits)
#pragma unroll
    for (int u = 0; u < PER; ++u) v[u] = v[u] + P[s * step + 256 * u];
  const int64_t m0 = (int64_t)tm * BM + (int)blockIdx.y * ROWS, n0 = (int64_t)tn * BM;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    const int i = threadIdx.x + 256 * u, r = i / BM, c = i % BM;
    if (m0 + r < e.M && n0 + c < e.N) {
      const T x = e.at(m0 + r, n0 + c, v[u]);
      *e.place(m0 + r, n0 + c) = x;
      if (mirror) turned[r][c] = x;
    }
  }
  if (mirror) {  // block-uniform
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = threadIdx.x + 256 * u, r = i % ROWS, c = i / ROWS;
      if (m0 + r < e.M && n0 + c < e.N) e.C[(n0 + c) * e.ldc + m0 + r] = turned[r][c];
    }
  }
  const int64_t n = n0 + threadIdx.x;
  if (a.dmode == kDColsum && tm == 0 && blockIdx.y == 0 && threadIdx.x < BM && n < k.N && k.D) {
    const T* S = (const T*)a.csws + (int64_t)blockIdx.x * BM + threadIdx.x;
    T x = S[0];
    for (int q = 1; q < a.splits; ++q) x = x + S[(int64_t)q * a.cut * BM];
    put_colsum(a, k, n, x);
  }
}

// Waves of a small-product block. More (gemm_direct_kernel takes 16) leave a wave 128
// registers, which the k-contiguous float32 loop spilled, and cost more in adding up their
// tiles than their shares of k saved: 512 k of 128 x 128, 9.7 us with 16.
constexpr int kGroupWaves = 8;

// Register q of a wave's tiles in LDS, [wave][regs][lane], added over the waves in order;
// all of them are read before the first is added.
template <typename T>
__device__ __forceinline__ T sum_waves(const T* __restrict__ part, int regs, int q, int lane, int nw) {
  T v[kGroupWaves];
#pragma unroll
  for (int w = 0; w < kGroupWaves; ++w) v[w] = w < nw ? part[(w * regs + q) * 64 + lane] : T(0);
  T s = v[0];
#pragma unroll
  for (int w = 1; w < kGroupWaves; ++w) s = s + v[w];
  return s;
}

// Small products: a 32 x 32 tile a block, k over its waves, whose partial tiles are
// added through LDS in wave order (gemm_direct_kernel for a group of tasks).
template <typename T, bool AKC, bool BKC>
__global__ void __launch_bounds__(64 * kGroupWaves) group_direct_kernel(GroupArgs a) {
  using MFT = MF<T>;
  using Dt = DirectTile<T>;
  constexpr int MT = MFT::MT, NACC = MFT::NACC, VEC = MFT::VEC, R = Dt::R, KB = Dt::KB, NCH = KB / 8;
  constexpr int CPT = kBKT<T> / 8;
  typedef typename MFT::vec_t VT;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  int ti, tm, tn;
  group_tile(a, 32, whole_tile(a, (int)blockIdx.x), ti, tm, tn);
  const GroupTask k = a.t[ti];
  const int64_t m0 = (int64_t)tm * 32, n0 = (int64_t)tn * 32;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = (int)(blockDim.x >> 6);
  const int g = lane / MT, c = lane % MT;
  const int Mp = pad_up(k.M, a.pad), Np = pad_up(k.N, a.pad), Kp = pad_up(k.K, a.pad);
  const int per = ((Kp + nw - 1) / nw + KB - 1) / KB * KB;  // a wave's k, whole batches
  const int kbeg = wave * per < Kp ? wave * per : Kp;
  const int kn = Kp - kbeg < per ? Kp - kbeg : per;
  typename MFT::acc_t acc[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = typename MFT::acc_t(0);
  const bool take_colsum = a.dmode == kDColsum && tm == 0 && k.D;
  double cs[R];
#pragma unroll
  for (int j = 0; j < R; ++j) cs[j] = 0.0;
  direct_product<T, AKC, BKC>(acc, (const T*)k.A, AKC ? Kp : Mp, Mp, m0, (const T*)k.B, BKC ? Kp : Np, Np, n0, kbeg, kn,
                              g, c, [&](const VT (&y)[R][NCH]) {
                                if (take_colsum) {
                                  // 16 k at a time in k order, the lane groups' shares by shuffle
#pragma unroll
                                  for (int j = 0; j < R; ++j)
#pragma unroll
                                    for (int c0 = 0; c0 < NCH; c0 += CPT) {
                                      T x = T(0);
#pragma unroll
                                      for (int ch = c0; ch < c0 + CPT; ++ch)
#pragma unroll
                                        for (int gg = 0; gg < MFT::G; ++gg)
#pragma unroll
                                          for (int q = 0; q < VEC; ++q) x = x + __shfl(y[j][ch][q], gg * MT + c, 64);
                                      cs[j] += (double)x;
                                    }
                                }
                              });
  T* part = reinterpret_cast<T*>(lds_raw);
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int r = 0; r < NACC; ++r) part[(wave * Dt::REGS + (i * R + j) * NACC + r) * 64 + lane] = acc[i][j][r];
  __syncthreads();
  const GroupEpi<T> e = group_epi<T>(a, k, a.sym && tm != tn);
  for (int q = wave; q < Dt::REGS; q += nw) {
    const T v = sum_waves(part, Dt::REGS, q, lane, nw);
    const int tt = q / NACC, r = q % NACC;
    const int64_t m = m0 + (tt / R) * MT + MFT::row(r, g), n = n0 + (tt % R) * MT + c;
    if (m < e.M && n < e.N) e.store(m, n, v);
  }
  if (take_colsum) {  // block-uniform; the waves' sums in order
    double* red = reinterpret_cast<double*>(lds_raw);
    __syncthreads();  // the partial tiles are read
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (g == 0) red[wave * 32 + j * MT + c] = cs[j];
    __syncthreads();
    for (int n = threadIdx.x; n < 32 && n0 + n < k.N; n += blockDim.x) {
      double x = red[n];
      for (int w = 1; w < nw; ++w) x += red[w * 32 + n];
      put_colsum(a, k, n0 + n, (T)x);
    }
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

// The same for few rows, or few columns: a 32 x 32 tile a block, as group_direct_kernel.
// A wave's lanes of one lane group hold MT columns of a row, so the statistics are
// butterflies over them and a part is MT columns wide.
template <typename T, bool BKC>
__global__ void __launch_bounds__(64 * kGroupWaves) stats_direct_kernel(StatsArgs a) {
  using MFT = MF<T>;
  using Dt = DirectTile<T>;
  constexpr int MT = MFT::MT, NACC = MFT::NACC, R = Dt::R, KB = Dt::KB, NCH = KB / 8;
  typedef typename MFT::vec_t VT;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int t = xcd_tile((int)blockIdx.x, a.tiles_m * a.tiles_n);
  int tm, tn;
  group_coords(t, a.tiles_m, a.tiles_n, 0, tm, tn);
  const int64_t m0 = (int64_t)tm * 32, n0 = (int64_t)tn * 32;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = (int)(blockDim.x >> 6);
  const int g = lane / MT, c = lane % MT;
  const int K = (int)a.K;
  const int per = ((K + nw - 1) / nw + KB - 1) / KB * KB;
  const int kbeg = wave * per < K ? wave * per : K;
  const int kn = K - kbeg < per ? K - kbeg : per;
  typename MFT::acc_t acc[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = typename MFT::acc_t(0);
  direct_product<T, true, BKC>(acc, (const T*)a.A, a.lda, a.M, m0, (const T*)a.B, a.ldb, a.N, n0, kbeg, kn, g, c,
                               [](const VT (&)[R][NCH]) {});
  T* part = reinterpret_cast<T*>(lds_raw);
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int r = 0; r < NACC; ++r) part[(wave * Dt::REGS + (i * R + j) * NACC + r) * 64 + lane] = acc[i][j][r];
  __syncthreads();
  T* C = (T*)a.C;
  for (int q = wave; q < Dt::REGS; q += nw) {
    const int tt = q / NACC, r = q % NACC, j = tt % R;
    const int64_t m = m0 + (tt / R) * MT + MFT::row(r, g), n = n0 + j * MT + c;
    // rows past the last are computed from it and not stored
    T z = sum_waves(part, Dt::REGS, q, lane, nw);
    const bool in = n < a.N;
    if (a.bias && in) z = z + ((const T*)a.bias)[n];
    if (!in) z = -INFINITY;
    T mx = z;
#pragma unroll
    for (int o = MT / 2; o >= 1; o >>= 1) mx = fmax(mx, __shfl_xor(mx, o, 64));
    T s = exp_of(z - (mx == -INFINITY ? T(0) : mx));
#pragma unroll
    for (int o = MT / 2; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if (m < a.M) {
      if (C && in) C[m * a.ldc + n] = z;
      if (a.targets && a.targets[m] == n) ((T*)a.zt)[m] = z;
      const int64_t p = (int64_t)tn * R + j;
      if (c == 0) {
        ((T*)a.pmax)[p * a.M + m] = mx;
        ((T*)a.psum)[p * a.M + m] = s;
      }
    }
  }
}

// Few rows (gemm_rows.h): a tile of 16 MR rows a block.
template <typename T, int MR, bool BKC>
__global__ void __launch_bounds__(64 * kRowsMaxWaves, (sizeof(T) == 4 && MR == 1 ? 4 : 2))
    group_rows_kernel(GroupArgs a) {
  using RT = RowsTile<T, BKC>;
  using RS = RowsSum<T, MR, BKC>;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = (int)(blockDim.x >> 6);
  const int first = lane < a.count ? a.first[lane] : 0x7fffffff;
  const int split = (int)blockIdx.x / a.tiles, b = (int)blockIdx.x - split * a.tiles;
  const int ti = __builtin_amdgcn_readfirstlane(63 - __builtin_clzll(__ballot(first <= b)));
  const GroupTask k = a.t[ti];
  const int tiles_m = (k.M + 16 * MR - 1) / (16 * MR);
  const int64_t m0 = (int64_t)((b - a.first[ti]) % tiles_m) * (16 * MR);
  const int64_t n0 = (int64_t)((b - a.first[ti]) / tiles_m) * RT::COLS;
  const int shares = nw * a.splits;  // of k
  const int per = ((k.K + shares - 1) / shares + RT::BATCH - 1) / RT::BATCH * RT::BATCH;
  const int64_t from = (int64_t)(split * nw + wave) * per;
  const int kbeg = from < k.K ? (int)from : k.K;
  const int kend = k.K - kbeg < per ? k.K : kbeg + per;
  RowsAcc<T> acc[MR][RT::NT];
#pragma unroll
  for (int i = 0; i < MR; ++i)
#pragma unroll
    for (int t = 0; t < RT::NT; ++t) acc[i][t] = RowsAcc<T>(0);
  rows_product<T, MR, BKC>(acc, (const T*)k.A, k.K, k.M, m0, (const T*)k.B, BKC ? k.K : k.N, k.N, n0, kbeg, kend, g, c);
  const RS sum{reinterpret_cast<T*>(lds_raw), lane, nw};
  sum.put(acc, wave);
  __syncthreads();
  if (a.splits > 1) {  // the raw partial
    T* P = (T*)a.ws + (int64_t)blockIdx.x * (RS::REGS * 64) + lane;
    for (int q = wave; q < RS::REGS; q += nw) P[q * 64] = sum.value(q);
    return;
  }
  const GroupEpi<T> e = group_epi<T>(a, k, false);
  for (int q = wave; q < RS::REGS; q += nw) {
    const int64_t m = m0 + 16 * (q / (4 * RT::NT)) + RowsMma<T>::row(q % 4, g), n = n0 + RT::col(c, q / 4 % RT::NT);
    const T v = sum.value(q);
    if (m < e.M && n < e.N) e.store(m, n, v);
  }
}

// The partials of a tile of few rows, added in split order, and the epilogue: block (v, y)
// takes four registers of tile v, a wave each.
template <typename T, int MR, bool BKC>
__global__ void __launch_bounds__(256) rows_sum_kernel(GroupArgs a) {
  using RT = RowsTile<T, BKC>;
  using RS = RowsSum<T, MR, BKC>;
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16, q = (int)blockIdx.y * 4 + (threadIdx.x >> 6);
  const int first = lane < a.count ? a.first[lane] : 0x7fffffff, b = (int)blockIdx.x;
  const int ti = __builtin_amdgcn_readfirstlane(63 - __builtin_clzll(__ballot(first <= b)));
  const GroupTask k = a.t[ti];
  const int tiles_m = (k.M + 16 * MR - 1) / (16 * MR);
  const int64_t m =
      (int64_t)((b - a.first[ti]) % tiles_m) * (16 * MR) + 16 * (q / (4 * RT::NT)) + RowsMma<T>::row(q % 4, g);
  const int64_t n = (int64_t)((b - a.first[ti]) / tiles_m) * RT::COLS + RT::col(c, q / 4 % RT::NT);
  const T* P = (const T*)a.ws + (int64_t)b * (RS::REGS * 64) + q * 64 + lane;
  const int64_t step = (int64_t)a.tiles * (RS::REGS * 64);
  T v = T(0);
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    T x[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = s0 + s < a.splits ? P[(s0 + s) * step] : T(0);
#pragma unroll
    for (int s = 0; s < 8; ++s) v = v + x[s];
  }
  const GroupEpi<T> e = group_epi<T>(a, k, false);
  if (m < e.M && n < e.N) e.store(m, n, v);
}

template <typename T, int MR, bool BKC>
__global__ void __launch_bounds__(64 * kRowsMaxWaves, (sizeof(T) == 4 && MR == 1 ? 4 : 2))
    stats_rows_kernel(StatsArgs a) {
  using RT = RowsTile<T, BKC>;
  using RS = RowsSum<T, MR, BKC>;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = (int)(blockDim.x >> 6);
  const int64_t m0 = (int64_t)((int)blockIdx.x % a.tiles_m) * (16 * MR);
  const int64_t p = (int)blockIdx.x / a.tiles_m, n0 = p * RT::COLS;
  const int K = (int)a.K, per = ((K + nw - 1) / nw + RT::BATCH - 1) / RT::BATCH * RT::BATCH;
  const int kbeg = wave * per < K ? wave * per : K;
  const int kend = kbeg + per < K ? kbeg + per : K;
  RowsAcc<T> acc[MR][RT::NT];
#pragma unroll
  for (int i = 0; i < MR; ++i)
#pragma unroll
    for (int t = 0; t < RT::NT; ++t) acc[i][t] = RowsAcc<T>(0);
  rows_product<T, MR, BKC>(acc, (const T*)a.A, a.lda, a.M, m0, (const T*)a.B, a.ldb, a.N, n0, kbeg, kend, g, c);
  const RS sum{reinterpret_cast<T*>(lds_raw), lane, nw};
  sum.put(acc, wave);
  __syncthreads();
  for (int u = wave; u < 4 * MR; u += nw) {  // the rows of registers r of row tile i: all their columns
    const int i = u / 4, r = u % 4;
    const int64_t m = m0 + 16 * i + RowsMma<T>::row(r, g);
    const int64_t tc = a.targets && m < a.M ? a.targets[m] : -1;
    T z[RT::NT], mx = -INFINITY, s = T(0);
#pragma unroll
    for (int t = 0; t < RT::NT; ++t) {
      const int64_t n = n0 + RT::col(c, t);
      T v = sum.value((i * RT::NT + t) * 4 + r);
      const bool in = n < a.N;
      if (a.bias && in) v = v + ((const T*)a.bias)[n];
      z[t] = in ? v : -INFINITY;
      mx = fmax(mx, z[t]);
      if (m < a.M) {
        if (a.C && in) ((T*)a.C)[m * a.ldc + n] = z[t];
        if (tc == n) ((T*)a.zt)[m] = z[t];
      }
    }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) mx = fmax(mx, __shfl_xor(mx, o, 64));
    const T ref = mx == -INFINITY ? T(0) : mx;
#pragma unroll
    for (int t = 0; t < RT::NT; ++t) s += exp_of(z[t] - ref);
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if (c == 0 && m < a.M) {
      ((T*)a.pmax)[p * a.M + m] = mx;
      ((T*)a.psum)[p * a.M + m] = s;
    }
  }
}

template <typename T, int BM>
void launch_group(const GroupArgs& a, int akc, int bkc, bool vec) {
  const unsigned grid = (unsigned)(a.cut * a.splits + a.tiles - a.cut);
  // Three blocks fit a CU by their LDS. Where the tasks' k differ, two: with three most
  // launches are placed at once, and no CU that is done early gets more (dw of 8 experts
  // as above, 305 -> 182 us; with equal k three are as good or better).
  const size_t lds = BM == 128 && !a.equal ? 56 * 1024 : kDmaLds<T, BM, BM> * sizeof(T);
#define DTMI_GROUP(AK, BKK)                                                  \
  if (vec)                                                                   \
    gemm_group_kernel<T, BM, AK, BKK, true><<<grid, 256, lds, stream()>>>(a);  \
  else                                                                       \
    gemm_group_kernel<T, BM, AK, BKK, false><<<grid, 256, lds, stream()>>>(a)
  if (akc && bkc) {
    DTMI_GROUP(true, true);
  } else if (akc) {
    DTMI_GROUP(true, false);
  } else {
    DTMI_GROUP(false, false);
  }
#undef DTMI_GROUP
  if (a.cut) group_sum_kernel<T, BM><<<dim3((unsigned)a.cut, BM * BM / 2048), 256, 0, stream()>>>(a);
}

template <typename T>
void launch_group_direct(const GroupArgs& a, int akc, int bkc, int nw) {
  size_t lds = (size_t)nw * DirectTile<T>::REGS * 64 * sizeof(T);  // the column sums' 32 doubles a wave fit in it
  const unsigned grid = (unsigned)a.tiles, th = 64u * (unsigned)nw;
  if (akc && bkc)
    group_direct_kernel<T, true, true><<<grid, th, lds, stream()>>>(a);
  else if (akc)
    group_direct_kernel<T, true, false><<<grid, th, lds, stream()>>>(a);
  else
    group_direct_kernel<T, false, false><<<grid, th, lds, stream()>>>(a);
}

template <typename T, int MR, bool BKC>
static void launch_rows_tile(const GroupArgs& a, int nw) {
  constexpr int REGS = RowsSum<T, MR, BKC>::REGS;
  group_rows_kernel<T, MR, BKC>
      <<<(unsigned)(a.tiles * a.splits), 64u * (unsigned)nw, (size_t)nw * REGS * 64 * sizeof(T), stream()>>>(a);
  if (a.splits > 1) rows_sum_kernel<T, MR, BKC><<<dim3((unsigned)a.tiles, REGS / 4), 256, 0, stream()>>>(a);
}

template <typename T>
void launch_group_rows(const GroupArgs& a, int bkc, int mr, int nw) {
  if (mr == 1)
    bkc ? launch_rows_tile<T, 1, true>(a, nw) : launch_rows_tile<T, 1, false>(a, nw);
  else
    bkc ? launch_rows_tile<T, 2, true>(a, nw) : launch_rows_tile<T, 2, false>(a, nw);
}

template <typename T>
void launch_stats_rows(const StatsArgs& a, int bkc, int mr, int nw) {
  const unsigned grid = (unsigned)(a.tiles_m * a.tiles_n), th = 64u * (unsigned)nw;
#define DTMI_ROWS(MR, BKK)                                                                      \
  stats_rows_kernel<T, MR, BKK><<<grid, th, (size_t)nw * RowsSum<T, MR, BKK>::REGS * 64 * sizeof(T), stream()>>>(a)
  if (mr == 1) {
    if (bkc)
      DTMI_ROWS(1, true);
    else
      DTMI_ROWS(1, false);
  } else {
    if (bkc)
      DTMI_ROWS(2, true);
    else
      DTMI_ROWS(2, false);
  }
#undef DTMI_ROWS
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

template <typename T>
void launch_stats_direct(const StatsArgs& a, int bkc, int nw) {
  const size_t lds = (size_t)nw * DirectTile<T>::REGS * 64 * sizeof(T);
  const unsigned grid = (unsigned)(a.tiles_m * a.tiles_n), th = 64u * (unsigned)nw;
  if (bkc)
    stats_direct_kernel<T, true><<<grid, th, lds, stream()>>>(a);
  else
    stats_direct_kernel<T, false><<<grid, th, lds, stream()>>>(a);
}

}  // namespace dtmi
