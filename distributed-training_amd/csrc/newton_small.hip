// Newton-Schulz steps of small and of thin matrices in the LDS of blocks of their own,
// where the grouped products (newton.hip) are 3 `steps` + 2 launches, each waiting for
// the one before.
// - Small: X, G and H of a matrix stay in one block from the norm to the result, one
//   launch a call.
// - Thin, of at most 64 rows or columns (float64 32; a block's share of X, G and H is then
//   too much to read and write for each step: 13 of 61 x 1362 as long as the groups) but too
//   many elements: a block for each 64 columns of X
//   takes a step on them and adds up their share of the next G; one block a matrix joins
//   the shares and forms H. 2 `steps` + 2 launches.
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
// 6 of 217 x 22 30 us, 16 of 64 x 64 36 us; float64, 6 of 64 x 64: 43 us. Thin,
// with its joins: 57 x 1124 16 us a step, 8 of 30 x 1000 in float64 12.
#include "newton_small.h"

#include <type_traits>

#include "gemm_rows.h"

namespace dtmi {

constexpr int kSmallTiles = 6;  // tiles of 16 rows: m up to 96
constexpr int kThinCols = 64;

__host__ __device__ inline int up16(int n) { return (n + 15) & ~15; }
// splits of the products G = X X^T along k
__host__ __device__ inline int small_splits(int pairs, int waves) { return pairs > waves / 2 ? 1 : waves / pairs; }

// A block's X [m, w], G and H in LDS. TM: most tiles of 16 rows, NW: waves.
template <typename T, int TM, int NW>
struct NewtonBlock {
  static constexpr int V = MF<T>::VEC, KB = 4 * V, TH = 64 * NW;
  typedef typename MF<T>::vec_t VT;
  using Acc = RowsAcc<T>;
  int mp, np, ldx, ldg, tiles, pairs, splits, per;
  // X's columns by 16, and the rows (of tiles) a wave takes of them
  int panels, height, shares;
  int lane, g, c, wave;
  T *X, *G, *H, *P;  // P: [pairs][splits][256] partial tiles

  __device__ __forceinline__ NewtonBlock(char* lds, int m, int w) {
    mp = up16(m);
    np = up16(w);
    ldx = np + V;
    ldg = mp + V;
    tiles = mp / 16;
    pairs = tiles * (tiles + 1) / 2;
    splits = small_splits(pairs, NW);
    per = (np / splits + KB - 1) / KB * KB;
    panels = np / 16;
    const int most = panels < NW ? NW / panels : 1;
    height = most >= tiles ? 1 : (tiles + most - 1) / most;
    shares = (tiles + height - 1) / height;
    lane = threadIdx.x & 63;
    g = lane / 16;
    c = lane % 16;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    X = reinterpret_cast<T*>(lds);
    G = X + mp * ldx;
    H = G + mp * ldg;
    P = H + mp * ldg;
  }
  __device__ __forceinline__ void clear() const {
    for (int i = threadIdx.x * V; i < mp * ldx; i += TH * V) *reinterpret_cast<VT*>(X + i) = VT(0);
  }
  // p = tm (tm + 1) / 2 + tn
  static __device__ __forceinline__ void pair(int p, int& tm, int& tn) {
    tm = 0;
    while ((tm + 1) * (tm + 2) / 2 <= p) ++tm;
    tn = p - tm * (tm + 1) / 2;
  }
  // rows 16 tm.. times rows 16 tn.. of R over kbeg <= k < kend
  __device__ __forceinline__ Acc product(const T* R, int ld, int tm, int tn, int kbeg, int kend) const {
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
  }
  // G = X X^T
  __device__ __forceinline__ void gram() const {
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
    if (splits == 1) return;
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
  // H = b G + c G G
  __device__ __forceinline__ void square(T cb, T cc) const {
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
  }
  // X = a X + H X: 16 columns a wave; fewer than the waves are shared by rows, and replaced
  // when all have been read
  __device__ __forceinline__ void apply(T ca) const {
    Acc acc[TM];
    auto read = [&](int u) {
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
      if (wave < panels * shares) read(wave);
      __syncthreads();
      if (wave < panels * shares) replace(wave);
    } else {
      for (int u = wave; u < panels; u += NW) {
        read(u);
        replace(u);
      }
    }
    __syncthreads();
  }
  // out[i] = gamma out[i] + rate X[at(i)], i < n
  template <typename AT>
  __device__ __forceinline__ void store(T* __restrict__ out, int n, T gamma, T rate, AT at) const {
    for (int i0 = threadIdx.x; i0 < n; i0 += 4 * TH) {
      T old[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) old[e] = gamma != T(0) && i0 + e * TH < n ? out[at.global(i0 + e * TH)] : T(0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e * TH;
        if (i < n) {
          const T x = rate * X[at.lds(i)];
          T* o = out + at.global(i);
          *o = gamma != T(0) ? fma(gamma, old[e], x) : x;
        }
      }
    }
  }
};

// Element i of columns c0 .. c0 + w of X (its rows, of a turned matrix): where it lies in
// the matrix [rows, cols] and in LDS.
struct NewtonAt {
  int64_t c0, cols;
  int w, ldx;
  bool tall;
  __device__ __forceinline__ int64_t global(int i) const {
    return tall ? c0 * cols + i : (int64_t)((unsigned)i / (unsigned)w) * cols + c0 + (unsigned)i % (unsigned)w;
  }
  __device__ __forceinline__ int lds(int i) const {
    const unsigned d = tall ? (unsigned)cols : (unsigned)w, q = (unsigned)i / d, r = (unsigned)i - q * d;
    return tall ? (int)r * ldx + (int)q : (int)q * ldx + (int)r;
  }
};

template <typename T, int TM, int NW>
__global__ void __launch_bounds__(64 * NW) newton_small_kernel(SmallArgs q) {
  using Block = NewtonBlock<T, TM, NW>;
  constexpr int V = Block::V, TH = Block::TH;
  typedef typename Block::VT VT;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  __shared__ double sh[NW];
  const SmallTask k = q.t[blockIdx.x];
  const bool tall = k.rows > k.cols;
  const Block x(lds_raw, tall ? k.cols : k.rows, tall ? k.rows : k.cols);
  const NewtonAt at{0, k.cols, tall ? k.rows : k.cols, x.ldx, tall};

  // u into X, and its sum of squares
  x.clear();
  __syncthreads();
  const T* __restrict__ U = (const T*)k.g;
  T* __restrict__ M = (T*)k.m;
  const T gs = q.gscale_dev ? (T)*q.gscale_dev : (T)q.gscale, mu = (T)q.mu;
  const int n = k.rows * k.cols;
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
        T v = u[e] * gs;
        if (M) {
          const T y = fma(mu, m[e], v);
          M[i] = y;
          v = q.nesterov ? fma(mu, y, v) : y;
        }
        x.X[at.lds(i)] = v;
        sq += (double)v * (double)v;
      }
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sq += __shfl_xor(sq, o, 64);
  if (x.lane == 0) sh[x.wave] = sq;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < NW; ++i) s += sh[i];
  const double scale = 1.0 / (sqrt(s) + q.eps);
  for (int i = threadIdx.x * V; i < x.mp * x.ldx; i += TH * V) {
    VT v = *reinterpret_cast<VT*>(x.X + i);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (T)((double)v[e] * scale);
    *reinterpret_cast<VT*>(x.X + i) = v;
  }
  __syncthreads();
  for (int step = 0; step < q.steps; ++step) {
    x.gram();
    x.square((T)q.b, (T)q.c);
    x.apply((T)q.a);
  }
  x.store((T*)k.out, n, (T)q.gamma, (T)k.rate, at);
}

// Thin matrices. Workspace of one: X by pieces of 64 columns [piece][mp][64], their shares
// of G [piece][mp][mp], H [mp][mp].
__host__ __device__ inline int64_t thin_pieces(int64_t w) { return (w + kThinCols - 1) / kThinCols; }

template <typename T, int TM, int NW>
__global__ void __launch_bounds__(64 * NW) newton_thin_kernel(ThinArgs q) {
  using Block = NewtonBlock<T, TM, NW>;
  constexpr int V = Block::V, TH = Block::TH;
  typedef typename Block::VT VT;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const int lane = threadIdx.x & 63;
  const int first = lane < q.count ? q.t[lane].first : 0x7fffffff;
  const int ti = __builtin_amdgcn_readfirstlane(63 - __builtin_clzll(__ballot(first <= (int)blockIdx.x)));
  const ThinTask k = q.t[ti];
  const bool tall = k.rows > k.cols;
  const int m = tall ? k.cols : k.rows, w = tall ? k.rows : k.cols, piece = (int)blockIdx.x - k.first;
  const int c0 = piece * kThinCols, cw = w - c0 < kThinCols ? w - c0 : kThinCols;
  const Block x(lds_raw, m, cw);
  const NewtonAt at{c0, k.cols, cw, x.ldx, tall};
  const int n = m * cw, square = x.mp * x.mp;
  T* Xg = (T*)k.ws + (int64_t)piece * (x.mp * kThinCols);
  T* Gg = (T*)k.ws + thin_pieces(w) * (x.mp * kThinCols) + (int64_t)piece * square;
  const T* Hg = (T*)k.ws + thin_pieces(w) * (x.mp * kThinCols + square);
  const int per_row = x.np / V, vectors = x.mp * per_row;
  if (q.stage == kThinFirst) {  // X = u / (|u| + eps), as norm_scale_kernel
    x.clear();
    double s = 0.0;
    const double* part = q.parts + (int64_t)(q.at + ti) * q.part_count;
    for (int i = lane; i < q.part_count; i += 64) s += part[i];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    const double scale = 1.0 / (sqrt(s) + q.eps);
    const T* U = (const T*)k.g;
    const T* M = (const T*)k.m;
    const T gs = q.gscale_dev ? (T)*q.gscale_dev : (T)q.gscale, mu = (T)q.mu;
    __syncthreads();
    for (int i0 = threadIdx.x; i0 < n; i0 += 4 * TH) {
      T u[4], v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = at.global(i0 + e * TH < n ? i0 + e * TH : 0);
        u[e] = U[i];
        v[e] = M ? M[i] : T(0);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e * TH;
        const T y = u[e] * gs, z = !M ? y : q.nesterov ? fma(mu, v[e], y) : v[e];
        if (i < n) x.X[at.lds(i)] = (T)((double)z * scale);
      }
    }
  } else {
    for (int i = threadIdx.x; i < vectors; i += TH) {
      const int r = i / per_row, v = (i - r * per_row) * V;
      *reinterpret_cast<VT*>(x.X + r * x.ldx + v) = *reinterpret_cast<const VT*>(Xg + r * kThinCols + v);
    }
    for (int i = threadIdx.x * V; i < square; i += TH * V) {
      const int r = i / x.mp;
      *reinterpret_cast<VT*>(x.H + r * x.ldg + (i - r * x.mp)) = *reinterpret_cast<const VT*>(Hg + i);
    }
    __syncthreads();
    x.apply((T)q.a);
    if (q.stage == kThinLast) {
      x.store((T*)k.out, n, (T)q.gamma, (T)k.rate, at);
      return;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < vectors; i += TH) {
    const int r = i / per_row, v = (i - r * per_row) * V;
    *reinterpret_cast<VT*>(Xg + r * kThinCols + v) = *reinterpret_cast<const VT*>(x.X + r * x.ldx + v);
  }
  x.gram();
  for (int i = threadIdx.x * V; i < square; i += TH * V) {
    const int r = i / x.mp;
    *reinterpret_cast<VT*>(Gg + i) = *reinterpret_cast<const VT*>(x.G + r * x.ldg + (i - r * x.mp));
  }
}

// G from its shares, in order, and H: one block a matrix.
template <typename T, int TM, int NW>
__global__ void __launch_bounds__(64 * NW) newton_thin_join_kernel(ThinArgs q) {
  using Block = NewtonBlock<T, TM, NW>;
  constexpr int V = Block::V, TH = Block::TH, U = 8;
  typedef typename Block::VT VT;
  extern __shared__ __attribute__((aligned(16))) char lds_raw[];
  const ThinTask k = q.t[blockIdx.x];
  const bool tall = k.rows > k.cols;
  const int m = tall ? k.cols : k.rows, w = tall ? k.rows : k.cols, pieces = (int)thin_pieces(w);
  const Block x(lds_raw, m, 16);
  const int square = x.mp * x.mp;
  const T* Gg = (const T*)k.ws + (int64_t)pieces * (x.mp * kThinCols);
  T* Hg = (T*)k.ws + (int64_t)pieces * (x.mp * kThinCols + square);
  for (int i = threadIdx.x * V; i < square; i += TH * V) {
    VT s = VT(0);
    for (int p0 = 0; p0 < pieces; p0 += U) {
      VT v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        v[u] = *reinterpret_cast<const VT*>(Gg + (int64_t)(p0 + u < pieces ? p0 + u : p0) * square + i);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p0 + u < pieces) s += v[u];
    }
    const int r = i / x.mp;
    *reinterpret_cast<VT*>(x.G + r * x.ldg + (i - r * x.mp)) = s;
  }
  __syncthreads();
  x.square((T)q.b, (T)q.c);
  for (int i = threadIdx.x * V; i < square; i += TH * V) {
    const int r = i / x.mp;
    *reinterpret_cast<VT*>(Hg + i) = *reinterpret_cast<const VT*>(x.H + r * x.ldg + (i - r * x.mp));
  }
}

// (by the most tiles a launch has)
constexpr int small_waves(int64_t tiles) { return tiles <= 2 || tiles > 4 ? 8 : 16; }

static int64_t lds_of(int dtype, int64_t m, int64_t w, int waves) {
  const int64_t es = dtype == DTMI_F32 ? 4 : 8, V = 16 / es, mp = up16((int)m), np = up16((int)w), t = mp / 16;
  const int64_t pairs = t * (t + 1) / 2, sp = small_splits((int)pairs, waves);
  return (mp * (np + V) + 2 * mp * (mp + V) + (sp > 1 ? pairs * sp * 256 : 0)) * es;
}

// The most tiles of 16 rows that a task has.
template <typename Task>
static int most_tiles(const Task* t, int count) {
  int tiles = 0;
  for (int i = 0; i < count; ++i) {
    const int n = (int)cdiv(t[i].rows < t[i].cols ? t[i].rows : t[i].cols, 16);
    tiles = n > tiles ? n : tiles;
  }
  return tiles;
}

int64_t small_lds(int dtype, int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols, w = rows < cols ? cols : rows;
  if (m > 16 * kSmallTiles || w > (1 << 16)) return INT64_MAX;
  return lds_of(dtype, m, w, 16);  // (the most splits)
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

int64_t thin_lds(int dtype, int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols, w = rows < cols ? cols : rows;
  return m > (dtype == DTMI_F32 ? 64 : 32) || w >= (1 << 20) ? INT64_MAX : lds_of(dtype, m, kThinCols, 16);
}

int64_t thin_bytes(int dtype, int64_t rows, int64_t cols) {
  const int64_t m = rows < cols ? rows : cols, w = rows < cols ? cols : rows, mp = up16((int)m);
  return ((thin_pieces(w) * (mp * kThinCols + mp * mp) + mp * mp) * (dtype == DTMI_F32 ? 4 : 8) + 255) / 256 * 256;
}

int64_t thin_blocks(int64_t rows, int64_t cols) { return thin_pieces(rows < cols ? cols : rows); }

double thin_cycles(int dtype, int64_t rows, int64_t cols, int64_t blocks, int64_t cus) {
  const int64_t m = rows < cols ? rows : cols, w = rows < cols ? cols : rows;
  const double t = (double)cdiv(m, 16), es = dtype == DTMI_F32 ? 4.0 : 8.0, mfma = dtype == DTMI_F32 ? 32.0 : 64.0;
  const double n = kThinCols / 16, pairs = t * (t + 1) / 2;
  const double step = 4.0 * (pairs * n + t * t * n) * mfma / 4.0 / 0.5;
  const double join = (double)thin_pieces(w) * 256.0 * t * t * es / 40.0 + 4.0 * pairs * t * mfma / 4.0 / 0.3;
  const double rounds = (double)blocks / (double)cus;
  return 22000.0 + step * (rounds > 1.0 ? rounds : 1.0) + join;
}

template <typename T, int TM>
static void launch_thin_tiles(const ThinArgs& a, int blocks, int64_t lds) {
  constexpr int NW = small_waves(TM);
  if (blocks)
    newton_thin_kernel<T, TM, NW><<<(unsigned)blocks, 64 * NW, (size_t)lds, stream()>>>(a);
  else
    newton_thin_join_kernel<T, TM, NW><<<(unsigned)a.count, 64 * NW, (size_t)lds, stream()>>>(a);
}

int launch_thin(int dtype, const ThinArgs& a, int blocks) {
  const int tiles = most_tiles(a.t, a.count);
  int64_t lds = 0;
  for (int i = 0; i < a.count; ++i) {
    const int64_t r = a.t[i].rows, c = a.t[i].cols;
    const int64_t l = lds_of(dtype, r < c ? r : c, kThinCols, small_waves(tiles));
    lds = l > lds ? l : lds;
  }
  if (dtype == DTMI_F64)
    launch_thin_tiles<double, 2>(a, blocks, lds);
  else if (tiles <= 2)
    launch_thin_tiles<float, 2>(a, blocks, lds);
  else
    launch_thin_tiles<float, 4>(a, blocks, lds);
  LAUNCH_CHECK("newton_thin_kernel");
  return DTMI_OK;
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
  const int tiles = most_tiles(a.t, count);
  int64_t lds = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t r = a.t[i].rows, c = a.t[i].cols;
    const int64_t l = lds_of(dtype, r < c ? r : c, r < c ? c : r, small_waves(tiles));
    lds = l > lds ? l : lds;
  }
  if (dtype == DTMI_F32)
    launch_type<float>(a, count, tiles, lds);
  else
    launch_type<double>(a, count, tiles, lds);
  LAUNCH_CHECK("newton_small_kernel");
  return DTMI_OK;
}

}  // namespace dtmi
