// Newton-Schulz steps of small matrices: X, G and H of one live in the LDS of one block
// from the norm to the result, so that a call is one launch where the grouped products
// (newton.hip) are 3 `steps` + 2 of them, each waiting for the one before.
//
// X is [m, w] with m <= w (a taller matrix is turned as it is read and written), m and w
// rounded up to 16 with zeros; the products run on 16 x 16 x 4 MFMAs, whose four k of a
// lane group are consecutive elements of a row: 16 bytes of LDS feed 4 (float64: 2) of
// them. Rows are 16 bytes longer than a multiple of 64: consecutive rows start in
// different banks.
//   G = X X^T        tiles on and below the diagonal, the waves sharing k where there are
//                    fewer than 8 of those
//   H = b G + c G G  likewise
//   X = a X + H X    a wave takes 16 columns, which nobody else reads, and replaces them;
//                    of few columns the waves share the rows
// Bound: the MFMAs of one CU and a few barriers a step. float32, five steps: 16 x 16 13 us,
// 6 of 217 x 22 30 us, 16 of 64 x 64 36 us; float64, 6 of 64 x 64: 43 us.
#include "newton_small.h"

#include <type_traits>

#include "gemm_rows.h"

namespace dtmi {

constexpr int kSmallTiles = 6;  // tiles of 16 rows: m up to 96

__host__ __device__ inline int up16(int n) { return (n + 15) & ~15; }
// splits of the products G = X X^T along k
__host__ __device__ inline int small_splits(int pairs, int waves) { return pairs > waves / 2 ? 1 : waves / pairs; }

// TM: most tiles of 16 rows, NW: waves.
template <typename T, int TM, int NW>
__global__ void __launch_bounds__(64 * NW) newton_small_kernel(SmallArgs q) {
  constexpr int V = MF<T>::VEC, KB = 4 * V, TH = 64 * NW;
  typedef typename MF<T>::vec_t VT;
  using Acc = RowsAcc<T>;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  __shared__ double sh[NW];
  const SmallTask k = q.t[blockIdx.x];
  const bool tall = k.rows > k.cols;
  const int mp = up16(tall ? k.cols : k.rows), np = up16(tall ? k.rows : k.cols);
  const int ldx = np + V, ldg = mp + V, tiles = mp / 16, pairs = tiles * (tiles + 1) / 2;
  T* X = reinterpret_cast<T*>(lds_raw);
  T* G = X + mp * ldx;
  T* H = G + mp * ldg;
  T* P = H + mp * ldg;  // [pairs][splits][256] partial tiles
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // u into X, and its sum of squares
  for (int i = threadIdx.x * V; i < mp * ldx; i += TH * V) *reinterpret_cast<VT*>(X + i) = VT(0);
  __syncthreads();
  const T* __restrict__ U = (const T*)k.g;
  T* __restrict__ M = (T*)k.m;
  const T gs = q.gscale_dev ? (T)*q.gscale_dev : (T)q.gscale, mu = (T)q.mu;
  const int n = k.rows * k.cols;
  auto at = [&](int i) {
    const int r = (int)((unsigned)i / (unsigned)k.cols), col = i - r * k.cols;
    return tall ? col * ldx + r : r * ldx + col;
  };
  double sq = 0.0;
  for (int i0 = threadIdx.x; i0 < n; i0 += 4 * TH) {  // four elements in flight
    T u[4], m[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e * TH;
      u[e] = i < n ? U[i] : T(0);
      m[e] = M && i < n ? M[i] : T(0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e * TH;
      if (i < n) {
        T x = u[e] * gs;
        if (M) {
          const T y = fma(mu, m[e], x);
          M[i] = y;
          x = q.nesterov ? fma(mu, y, x) : y;
        }
        X[at(i)] = x;
        sq += (double)x * (double)x;
      }
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sq += __shfl_xor(sq, o, 64);
  if (lane == 0) sh[wave] = sq;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < NW; ++i) s += sh[i];
  const double scale = 1.0 / (sqrt(s) + q.eps);
  for (int i = threadIdx.x * V; i < mp * ldx; i += TH * V) {
    VT v = *reinterpret_cast<VT*>(X + i);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)((double)v[e] * scale);
    *reinterpret_cast<VT*>(X + i) = v;
  }
  __syncthreads();

  auto pair = [&](int p, int& tm, int& tn) {  // p = tm (tm + 1) / 2 + tn
    tm = 0;
    while ((tm + 1) * (tm + 2) / 2 <= p) ++tm;
    tn = p - tm * (tm + 1) / 2;
  };
  // rows 16 tm.. times rows 16 tn.. of R over kbeg <= k < kend
  auto product = [&](const T* R, int ld, int tm, int tn, int kbeg, int kend) {
    Acc acc = Acc(0);
    const T* a = R + (16 * tm + c) * ld + V * g;
    const T* b = R + (16 * tn + c) * ld + V * g;
    auto some = [&](auto count, int kk) {  // their loads first: few waves hide each other's
      constexpr int N = decltype(count)::value;
      VT va[N], vb[N];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        va[u] = *reinterpret_cast<const VT*>(a + kk + u * KB);
        vb[u] = *reinterpret_cast<const VT*>(b + kk + u * KB);
      }
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) acc = RowsMma<T>::mma(va[u][e], vb[u][e], acc);
    };
    constexpr int DEEP = TM == kSmallTiles ? 2 : 4;
    int kk = kbeg;
    for (; kk + (DEEP - 1) * KB < kend; kk += DEEP * KB) some(std::integral_constant<int, DEEP>(), kk);
    for (; kk < kend; kk += KB) some(std::integral_constant<int, 1>(), kk);
    return acc;
  };
  const int splits = small_splits(pairs, NW), per = (np / splits + KB - 1) / KB * KB;
  // X's columns by 16, and the rows (of tiles) a wave takes of them
  const int panels = np / 16, most = panels < NW ? NW / panels : 1;
  const int height = most >= tiles ? 1 : (tiles + most - 1) / most, shares = (tiles + height - 1) / height;
  const T ca = (T)q.a, cb = (T)q.b, cc = (T)q.c;
  for (int step = 0; step < q.steps; ++step) {
    for (int u = wave; u < pairs * splits; u += NW) {
      int tm, tn;
      pair(u / splits, tm, tn);
      const int kbeg = u % splits * per, kend = u % splits + 1 == splits ? np : kbeg + per;
      const Acc acc = product(X, ldx, tm, tn, kbeg < np ? kbeg : np, kend < np ? kend : np);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * tm + RowsMma<T>::row(r, g), col = 16 * tn + c;
        if (splits > 1) {
          P[u * 256 + r * 64 + lane] = acc[r];
        } else {
          G[row * ldg + col] = acc[r];
          if (tm != tn) G[col * ldg + row] = acc[r];
        }
      }
    }
    __syncthreads();
    if (splits > 1) {
      for (int i = threadIdx.x; i < pairs * 256; i += TH) {
        int tm, tn;
        pair(i / 256, tm, tn);
        const T* p = P + (i / 256) * splits * 256 + i % 256;
        T v = p[0];
        for (int w = 1; w < splits; ++w) v += p[w * 256];
        const int row = 16 * tm + RowsMma<T>::row(i % 256 / 64, g), col = 16 * tn + c;
        G[row * ldg + col] = v;
        if (tm != tn) G[col * ldg + row] = v;
      }
      __syncthreads();
    }
    for (int u = wave; u < pairs; u += NW) {
      int tm, tn;
      pair(u, tm, tn);
      const Acc acc = product(G, ldg, tm, tn, 0, mp);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * tm + RowsMma<T>::row(r, g), col = 16 * tn + c;
        const T h = fma(cb, G[row * ldg + col], cc * acc[r]);
        H[row * ldg + col] = h;
        if (tm != tn) H[col * ldg + row] = h;
      }
    }
    __syncthreads();
    // 16 columns a wave; fewer than the waves are shared by rows, and replaced when all
    // have been read
    Acc acc[TM];
    auto apply = [&](int u) {
      const T* x = X + 16 * (u % panels) + c;
      const T* h = H + (16 * (u / panels * height) + c) * ldg + V * g;
      const int count = tiles - u / panels * height < height ? tiles - u / panels * height : height;
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[i] = Acc(0);
      for (int kk = 0; kk < mp; kk += KB) {
        T b[V];
#pragma unroll
        for (int e = 0; e < V; ++e) b[e] = x[(kk + V * g + e) * ldx];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          if (i < count) {
            const VT a = *reinterpret_cast<const VT*>(h + 16 * i * ldg + kk);
#pragma unroll
            for (int e = 0; e < V; ++e) acc[i] = RowsMma<T>::mma(a[e], b[e], acc[i]);
          }
        }
      }
    };
    auto replace = [&](int u) {
      T* x = X + 16 * (u / panels * height) * ldx + 16 * (u % panels) + c;
      const int count = tiles - u / panels * height < height ? tiles - u / panels * height : height;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if (i < count) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            T* y = x + (16 * i + RowsMma<T>::row(r, g)) * ldx;
            *y = fma(ca, *y, acc[i][r]);
          }
        }
      }
    };
    if (height < tiles) {
      if (wave < panels * shares) apply(wave);
      __syncthreads();
      if (wave < panels * shares) replace(wave);
    } else {
      for (int u = wave; u < panels; u += NW) {
        apply(u);
        replace(u);
      }
    }
    __syncthreads();
  }
  T* __restrict__ out = (T*)k.out;
  const T gamma = (T)q.gamma, rate = (T)k.rate;
  for (int i0 = threadIdx.x; i0 < n; i0 += 4 * TH) {
    T old[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) old[e] = gamma != T(0) && i0 + e * TH < n ? out[i0 + e * TH] : T(0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + e * TH;
      if (i < n) {
        const T x = rate * X[at(i)];
        out[i] = gamma != T(0) ? fma(gamma, old[e], x) : x;
      }
    }
  }
}

// (by the most tiles a launch has)
constexpr int small_waves(int64_t tiles) { return tiles <= 2 || tiles > 4 ? 8 : 16; }

static int64_t lds_of(int dtype, int64_t rows, int64_t cols, int waves) {
  const int64_t m = rows < cols ? rows : cols, w = rows < cols ? cols : rows;
  const int64_t es = dtype == DTMI_F32 ? 4 : 8, V = 16 / es, mp = up16((int)m), np = up16((int)w), t = mp / 16;
  const int64_t pairs = t * (t + 1) / 2, sp = small_splits((int)pairs, waves);
  return (mp * (np + V) + 2 * mp * (mp + V) + (sp > 1 ? pairs * sp * 256 : 0)) * es;
}

int64_t small_lds(int dtype, int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols, w = rows < cols ? cols : rows;
  if (m > 16 * kSmallTiles || w > (1 << 16)) return INT64_MAX;
  return lds_of(dtype, rows, cols, 16);  // (the most splits)
}

double small_cycles(int dtype, int64_t rows, int64_t cols, int steps) {
  const int64_t m = rows < cols ? rows : cols, w = rows < cols ? cols : rows;
  const double t = (double)cdiv(m, 16), n = (double)cdiv(w, 16), pairs = t * (t + 1) / 2;
  // 4 MFMAs a tile and 16 k, on four SIMDs
  const double mma = 4.0 * (pairs * n + pairs * t + t * t * n) * (dtype == DTMI_F32 ? 32.0 : 64.0) / 4.0;
  return 20000.0 + steps * (4000.0 + mma / 0.5);
}

int64_t small_lds_limit() {
  static const int64_t limit = [] {
    int dev = 0, v = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&v, hipDeviceAttributeMaxSharedMemoryPerBlock, dev) != hipSuccess)
      v = 0;
    return (int64_t)v - 256;  // the kernel's own
  }();
  return limit;
}

template <typename T, int TM>
static void launch_tiles(const SmallArgs& a, int count, int64_t lds) {
  constexpr int NW = small_waves(TM);
  newton_small_kernel<T, TM, NW><<<(unsigned)count, 64 * NW, (size_t)lds, stream()>>>(a);
}

template <typename T>
static void launch_type(const SmallArgs& a, int count, int tiles, int64_t lds) {
  if (tiles <= 2)
    launch_tiles<T, 2>(a, count, lds);
  else if (tiles <= 4)
    launch_tiles<T, 4>(a, count, lds);
  else
    launch_tiles<T, kSmallTiles>(a, count, lds);
}

int launch_small(int dtype, const SmallArgs& a, int count) {
  int64_t lds = 0, tiles = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t m = a.t[i].rows < a.t[i].cols ? a.t[i].rows : a.t[i].cols;
    tiles = cdiv(m, 16) > tiles ? cdiv(m, 16) : tiles;
  }
  for (int i = 0; i < count; ++i) {
    const int64_t l = lds_of(dtype, a.t[i].rows, a.t[i].cols, small_waves(tiles));
    lds = l > lds ? l : lds;
  }
  if (dtype == DTMI_F32)
    launch_type<float>(a, count, (int)tiles, lds);
  else
    launch_type<double>(a, count, (int)tiles, lds);
  LAUNCH_CHECK("newton_small_kernel");
  return DTMI_OK;
}

}  // namespace dtmi
