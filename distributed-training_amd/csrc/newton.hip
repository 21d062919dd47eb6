// Orthogonalised updates: Newton-Schulz steps on the singular values of a set of
// matrices, and the optimizer step made of them.
//
//   X = U / (|U|_F + eps);  `steps` times: G = X X^T, H = b G + c G G, X = a X + H X
//
// for a matrix of no more rows than columns; a taller one is worked on transposed, from
// the pass that scales it to the last product, which writes it back the other way
// round. G and H are symmetric: their products run over the tiles on and below the
// diagonal and mirror the rest, so that a step of an m x n matrix (m <= n) costs m^2 n
// + m^3 + 2 m^2 n operations, a third less than three plain products where m = n. All
// matrices of a call share each launch (gemm_group.h).
// Bound: MFMA; small matrices by 3 `steps` launches one after the other, but for those of
// newton_small.hip.
#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "gemm_group.h"
#include "newton_small.h"
#include "seqmath.h"

namespace dtmi {

constexpr int kNormTasks = 56;  // 56 bytes each: the arguments stay below 4 KB

// X is [rows, cols], or [cols, rows] of a matrix with more rows than columns, with both
// rounded up to 16 bytes of elements and zeros there.
struct NormTask {
  const void* g;
  void* m;  // momentum (NULL: u = g)
  void* x;  // u / (|u| + eps)
  double* part;  // [parts]
  int rows, cols;
};

struct NormArgs {
  int nesterov, parts;
  double mu, eps, gscale;
  const double* gscale_dev;
  NormTask t[kNormTasks];
};

// The step's u of V elements from element i on; m moved on where FIRST.
template <typename T, int V, bool FIRST>
__device__ __forceinline__ void norm_u(T (&u)[V], const NormArgs& a, const T* __restrict__ G, T* __restrict__ M,
                                       int64_t i, T gs, T mu) {
  vload<T, V>(u, G + i);
#pragma unroll
  for (int e = 0; e < V; ++e) u[e] = u[e] * gs;
  if (!M) return;
  T m[V];
  vload<T, V>(m, M + i);
  if constexpr (FIRST) {
#pragma unroll
    for (int e = 0; e < V; ++e) m[e] = fma(mu, m[e], u[e]);
    vstore<T, V>(M + i, m);
  }
#pragma unroll
  for (int e = 0; e < V; ++e) u[e] = a.nesterov ? fma(mu, m[e], u[e]) : m[e];
}

// m = mu m + g, and the block's share of the sum of squares of u = g + mu m (nesterov)
// or m, in float64.
template <typename T>
__global__ void __launch_bounds__(256) norm_sum_kernel(NormArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  const NormTask k = a.t[blockIdx.y];
  const T* G = (const T*)k.g;
  T* M = (T*)k.m;
  const T gs = a.gscale_dev ? (T)*a.gscale_dev : (T)a.gscale, mu = (T)a.mu;
  const int64_t n = (int64_t)k.rows * k.cols, stride = (int64_t)gridDim.x * 256;
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t nv = aligned(G, 16) && aligned(M, 16) ? n / V : 0;
  double sq = 0.0;
  int64_t v = first;
  for (; v + 3 * stride < nv; v += 4 * stride) {  // four vectors in flight
    T u[4][V];
#pragma unroll
    for (int q = 0; q < 4; ++q) norm_u<T, V, true>(u[q], a, G, M, (v + q * stride) * V, gs, mu);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < V; ++e) sq += (double)u[q][e] * (double)u[q][e];
  }
  for (; v < nv; v += stride) {
    T u[V];
    norm_u<T, V, true>(u, a, G, M, v * V, gs, mu);
#pragma unroll
    for (int e = 0; e < V; ++e) sq += (double)u[e] * (double)u[e];
  }
  for (int64_t i = nv * V + first; i < n; i += stride) {
    T u[1];
    norm_u<T, 1, true>(u, a, G, M, i, gs, mu);
    sq += (double)u[0] * (double)u[0];
  }
  __shared__ double sh[4];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) sq += __shfl_xor(sq, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sq;
  __syncthreads();
  if (threadIdx.x == 0) k.part[blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// X = u / (|u| + eps), u formed again from g and m: written by the first pass it would be
// read here just the same. The padding of X is set to 0.
template <typename T>
__global__ void __launch_bounds__(256) norm_scale_kernel(NormArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  const NormTask k = a.t[blockIdx.y];
  const T* G = (const T*)k.g;
  T* M = (T*)k.m;
  T* X = (T*)k.x;
  const T gs = a.gscale_dev ? (T)*a.gscale_dev : (T)a.gscale, mu = (T)a.mu;
  double s = 0.0;  // every wave adds the parts in the same order
  for (int i = threadIdx.x & 63; i < a.parts; i += 64) s += k.part[i];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  const double scale = 1.0 / (sqrt(s) + a.eps);
  if (k.rows > k.cols) {  // block-uniform: 32 x 32 pieces turned through LDS
    __shared__ T turned[32][33];
    const uint32_t pr = (uint32_t)((k.rows + V - 1) / V * V), pc = (uint32_t)((k.cols + V - 1) / V * V);
    const uint32_t across = (pc + 31) / 32, pieces = across * ((pr + 31) / 32);
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
      const uint32_t r0 = p / across * 32, c0 = p % across * 32;
#pragma unroll
      for (int y = ty; y < 32; y += 8) {
        const uint32_t r = r0 + y, c = c0 + tx;
        T u[1] = {T(0)};
        const bool in = r < (uint32_t)k.rows && c < (uint32_t)k.cols;
        if (in) norm_u<T, 1, false>(u, a, G, M, (int64_t)r * k.cols + c, gs, mu);
        turned[y][tx] = in ? (T)((double)u[0] * scale) : T(0);
      }
      __syncthreads();
#pragma unroll
      for (int y = ty; y < 32; y += 8) {
        const uint32_t c = c0 + y, r = r0 + tx;
        if (c < pc && r < pr) X[(int64_t)c * pr + r] = turned[tx][y];
      }
      __syncthreads();
    }
    return;
  }
  const uint32_t per_row = (uint32_t)((k.cols + V - 1) / V);
  const uint32_t rows = (uint32_t)((k.rows + V - 1) / V * V), total = rows * per_row;
  const bool vec = aligned(G, 16) && aligned(M, 16) && k.cols % V == 0;
  for (uint32_t v = blockIdx.x * 256 + threadIdx.x; v < total; v += gridDim.x * 256) {
    const uint32_t r = v / per_row, c = (v - r * per_row) * V;
    T x[V];
    if (r >= (uint32_t)k.rows) {
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = T(0);
    } else if (vec) {
      norm_u<T, V, false>(x, a, G, M, (int64_t)r * k.cols + c, gs, mu);
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = (T)((double)x[e] * scale);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        T u[1] = {T(0)};
        if (c + e < (uint32_t)k.cols) norm_u<T, 1, false>(u, a, G, M, (int64_t)r * k.cols + c + e, gs, mu);
        x[e] = (T)((double)u[0] * scale);
        if (c + e >= (uint32_t)k.cols) x[e] = T(0);
      }
    }
    vstore<T, V>(X + (int64_t)v * V, x);
  }
}

struct NewtonArgs {
  int n, steps, nesterov;
  const void* const* g;
  void* const* m;    // momenta, or NULL
  void* const* out;  // where the result goes
  const int64_t* rows;
  const int64_t* cols;
  double a, b, c, eps, mu, gscale;
  const double* gscale_dev;
  // out = gamma out + rate[i] X (rate NULL: out = X)
  double gamma;
  const double* rate;
};

// Blocks per matrix of the norm kernels, by the largest one's elements: a vector a thread
// up to `most` blocks.
static int norm_blocks(int64_t elements, size_t es, int most) {
  const int64_t p = cdiv(elements * (int64_t)es, 16 * 256);
  return (int)(p < 1 ? 1 : p > most ? most : p);
}

static int64_t up(int64_t n, int64_t v) { return cdiv(n, v) * v; }
static size_t bytes_of(int64_t r, int64_t c, size_t es) {
  const int64_t v = 16 / (int64_t)es;
  return ((size_t)up(r, v) * up(c, v) * es + 255) & ~(size_t)255;
}

// The sums of squares of all u, momenta moved on, and, with x, u / (|u| + eps) there.
template <typename T>
static int norms(const NewtonArgs& q, const std::vector<int>& live, int64_t most, int np, double* parts,
                 const std::vector<char*>* x) {
  const int n = (int)live.size();
  for (int lo = 0; lo < n; lo += kNormTasks) {
    NormArgs a{};
    const int count = n - lo < kNormTasks ? n - lo : kNormTasks;
    a.nesterov = q.nesterov;
    a.parts = np;
    a.mu = q.mu;
    a.eps = q.eps;
    a.gscale = q.gscale;
    a.gscale_dev = q.gscale_dev;
    double bytes = 0;
    for (int i = 0; i < count; ++i) {
      const int j = live[lo + i];
      a.t[i] = {q.g[j], q.m ? q.m[j] : nullptr, x ? (*x)[lo + i] : nullptr, parts + (size_t)(lo + i) * np, (int)q.rows[j],
                (int)q.cols[j]};
      bytes += (double)q.rows[j] * (double)q.cols[j] * (double)sizeof(T) * (x ? (q.m ? 6 : 3) : (q.m ? 3 : 1));
    }
    TimedLaunch tl(DTMI_FAM_OTHER, bytes);
    norm_sum_kernel<T><<<dim3((unsigned)np, (unsigned)count), 256, 0, stream()>>>(a);
    const int blocks = norm_blocks(most, sizeof(T), 4096 / count < 64 ? 64 : 4096 / count);
    if (x) norm_scale_kernel<T><<<dim3((unsigned)blocks, (unsigned)count), 256, 0, stream()>>>(a);
    LAUNCH_CHECK("norm kernels");
  }
  return DTMI_OK;
}

template <typename T>
static int newton_run(int dtype, const NewtonArgs& q, const std::vector<int>& live, int64_t most, int np, char* ws) {
  constexpr size_t es = sizeof(T);
  // The workspace's matrices are padded to 16 bytes of elements both ways, with zeros, so
  // that odd sizes run on 16-byte loads too: zero rows and columns stay zero through the
  // steps. The last product writes the result as it lies.
  constexpr int V = 16 / (int)sizeof(T);
  const int n = (int)live.size();
  std::vector<char*> x0(n), x1(n), G(n), H(n);
  double* parts = (double*)ws;
  char* p = ws + (((size_t)n * np * sizeof(double) + 255) & ~(size_t)255);
  for (int i = 0; i < n; ++i) {
    const int64_t r = q.rows[live[i]], c = q.cols[live[i]], s = r < c ? r : c;
    const size_t xb = bytes_of(r, c, es), gb = bytes_of(s, s, es);
    x0[i] = p;
    x1[i] = p + xb;
    G[i] = p + 2 * xb;
    H[i] = G[i] + gb;
    p = H[i] + gb;
  }
  int rc = norms<T>(q, live, most, np, parts, &x0);
  if (rc) return rc;
  // the launches of a step from x0 to x1 and of one from x1 to x0, and of the last
  std::vector<GroupTask> t(n);
  std::vector<GroupLaunch> gram[2], sq, apply[2], final;
  auto of = [&](int i, int& m, int& w) {
    const int64_t r = q.rows[live[i]], c = q.cols[live[i]];
    m = (int)(r < c ? r : c);
    w = (int)(r < c ? c : r);
    return r > c;
  };
  int m, w;
  for (int i = 0; i < n; ++i) {  // H = b G + c G G (G = G^T)
    of(i, m, w);
    t[i] = {G[i], G[i], H[i], G[i], m, m, m, 0, 1.0};
  }
  rc = plan_group(dtype, 1, 1, t, kDMatrix, 1, q.c, q.b, 0.0, V, V, sq);
  for (int odd = 0; odd < 2 && odd < q.steps && !rc; ++odd) {
    for (int i = 0; i < n; ++i) {  // G = X X^T
      of(i, m, w);
      t[i] = {x0[i], x0[i], G[i], nullptr, m, m, w, 0, 1.0};
    }
    rc = plan_group(dtype, 1, 1, t, kDNone, 1, 1.0, 0.0, 0.0, V, V, gram[odd]);
    const bool ends = (q.steps - 1) % 2 == odd;
    for (int end = 0; end < 2 && !rc; ++end) {  // X = a X + H X, the last into the result
      if (end ? !ends : q.steps < odd + 2) continue;
      for (int i = 0; i < n; ++i) {
        const bool tall = of(i, m, w);
        t[i] = {H[i], x0[i], end ? (char*)q.out[live[i]] : x1[i], x0[i], m, w, m, end && tall,
                end && q.rate ? q.rate[live[i]] : 1.0};
      }
      rc = plan_group(dtype, 1, 0, t, kDMatrix, 0, 1.0, q.a, end && q.rate ? q.gamma : 0.0, V, end ? 1 : V,
                      end ? final : apply[odd]);
    }
    std::swap(x0, x1);
  }
  for (int s = 0; s < q.steps && !rc; ++s) {
    rc = launch_group(dtype, gram[s % 2]);
    if (!rc) rc = launch_group(dtype, sq);
    if (!rc) rc = launch_group(dtype, s + 1 == q.steps ? final : apply[s % 2]);
  }
  return rc;
}

// How to run a call: by the least of what the three ways are estimated to take, in cycles.
// Small and thin matrices (newton_small.hip) are so only all together: beside others they
// cost the groups no launch. float32, five steps, microseconds:
//                    small  thin  groups                     small  thin  groups
//   16 x 16             13           80    2 of 1102 x 41             76   144
//   15 of 35 x 264      51          115    48 of 64 x 768            163   182
//   8 of 96 x 96        80           98    16 of 64 x 8192           394   297
//   8 of 96 x 192      119           99    float64, 8 of 30 x 1000    70   172
// A group's launch takes about 7 us whatever its size.
enum NewtonWay { kSmall, kThin, kGroups };
static NewtonWay newton_way(int dtype, const NewtonArgs& q, const std::vector<int>& live, size_t& thin_ws) {
  const int64_t cus = num_cus() > 0 ? num_cus() : 256, limit = small_lds_limit();
  const double never = 1e200, launches = (double)cdiv((int64_t)live.size(), kSmallTasks);
  double small = 0, thin = 0, operations = 0;
  int64_t blocks = 0;
  thin_ws = 256;
  for (int i : live) {
    const int64_t r = q.rows[i], c = q.cols[i];
    const double m = (double)(r < c ? r : c), w = (double)(r < c ? c : r);
    operations += q.steps * (3.0 * m * m * w + m * m * m);
    small = small_lds(dtype, r, c) > limit ? never : std::max(small, small_cycles(dtype, r, c, q.steps));
    if (thin_lds(dtype, r, c) > limit) thin = never;
    if (thin == never) continue;
    blocks += thin_blocks(r, c);
    thin_ws += thin_bytes(dtype, r, c);
  }
  if (blocks >= 1 << 24) thin = never;
  for (int i : live)
    if (thin != never) thin = std::max(thin, thin_cycles(dtype, q.rows[i], q.cols[i], blocks, cus));
  const double rate = (dtype == DTMI_F32 ? 256.0 : 128.0) * (double)cus;
  const double groups = 3.0 * q.steps * 17000.0 + operations / rate;
  small *= launches;
  thin = launches * (25000.0 + q.steps * thin);
  return small <= thin && small < groups ? kSmall : thin < groups ? kThin : kGroups;
}

static int run_small(int dtype, const NewtonArgs& q, const std::vector<int>& live) {
  const double es = dtype == DTMI_F32 ? 4.0 : 8.0;
  for (size_t lo = 0; lo < live.size(); lo += kSmallTasks) {
    SmallArgs a{};
    const size_t count = live.size() - lo < kSmallTasks ? live.size() - lo : kSmallTasks;
    a.steps = q.steps;
    a.nesterov = q.nesterov;
    a.a = q.a;
    a.b = q.b;
    a.c = q.c;
    a.eps = q.eps;
    a.mu = q.mu;
    a.gscale = q.gscale;
    a.gscale_dev = q.gscale_dev;
    a.gamma = q.rate ? q.gamma : 0.0;
    double bytes = 0;
    for (size_t i = 0; i < count; ++i) {
      const int j = live[lo + i];
      a.t[i] = {q.g[j], q.m ? q.m[j] : nullptr, q.out[j], q.rate ? q.rate[j] : 1.0, (int)q.rows[j], (int)q.cols[j]};
      bytes += (double)q.rows[j] * (double)q.cols[j] * es * (q.m ? 5 : 2);
    }
    TimedLaunch tl(DTMI_FAM_OTHER, bytes);
    const int rc = launch_small(dtype, a, (int)count);
    if (rc) return rc;
  }
  return DTMI_OK;
}

template <typename T>
static int run_thin(int dtype, const NewtonArgs& q, const std::vector<int>& live, int64_t most, int np, char* ws) {
  double* parts = (double*)ws;
  char* p = ws + ((live.size() * (size_t)np * sizeof(double) + 255) & ~(size_t)255);
  int rc = norms<T>(q, live, most, np, parts, nullptr);
  for (size_t lo = 0; lo < live.size() && !rc; lo += kSmallTasks) {
    ThinArgs a{};
    a.count = live.size() - lo < kSmallTasks ? (int)(live.size() - lo) : kSmallTasks;
    a.nesterov = q.nesterov;
    a.at = (int)lo;
    a.part_count = np;
    a.parts = parts;
    a.a = q.a;
    a.b = q.b;
    a.c = q.c;
    a.eps = q.eps;
    a.mu = q.mu;
    a.gscale = q.gscale;
    a.gscale_dev = q.gscale_dev;
    a.gamma = q.rate ? q.gamma : 0.0;
    int64_t blocks = 0;
    double operations = 0;
    for (int i = 0; i < a.count; ++i) {
      const int j = live[lo + i];
      const int64_t r = q.rows[j], c = q.cols[j];
      const double m = (double)(r < c ? r : c), w = (double)(r < c ? c : r);
      a.t[i] = {q.g[j], q.m ? q.m[j] : nullptr, q.out[j], p, q.rate ? q.rate[j] : 1.0, (int)r, (int)c, (int)blocks};
      p += thin_bytes(dtype, r, c);
      blocks += thin_blocks(r, c);
      operations += q.steps * (3.0 * m * m * w + m * m * m);
    }
    TimedLaunch tl(DTMI_FAM_GEMM, operations);
    a.stage = kThinFirst;
    rc = launch_thin(dtype, a, (int)blocks);
    for (int s = 0; s < q.steps && !rc; ++s) {
      rc = launch_thin(dtype, a, 0);
      a.stage = s + 1 == q.steps ? kThinLast : kThinStep;
      if (!rc) rc = launch_thin(dtype, a, (int)blocks);
    }
  }
  return rc;
}

static int newton(const char* what, int dtype, const NewtonArgs& q) {
  DTMI_CHECK(q.n >= 0 && q.steps >= 1 && q.steps <= 64, "%s: needs 1 to 64 steps, not %d", what, q.steps);
  DTMI_CHECK(q.n == 0 || (q.g && q.out && q.rows && q.cols), "%s: NULL array", what);
  const size_t es = dtype == DTMI_F32 ? 4 : 8;
  std::vector<int> live;
  size_t bytes = 256;
  int64_t most = 0;
  for (int i = 0; i < q.n; ++i) {
    const int64_t r = q.rows[i], c = q.cols[i], edge = (1 << 24) / (int64_t)es - 4;
    DTMI_CHECK(r >= 0 && c >= 0, "%s: negative size of matrix %d", what, i);
    if (r == 0 || c == 0) continue;
    DTMI_CHECK(r < edge && c < edge && up(r, 4) * up(c, 4) < (1LL << 32),
               "%s: matrix %d, %lld x %lld, is too large (rows and columns below 2^24 bytes, 2^32 elements)", what, i,
               (long long)r, (long long)c);
    DTMI_CHECK(q.g[i] && q.out[i] && (!q.m || q.m[i]), "%s: NULL pointer of matrix %d", what, i);
    const int64_t s = r < c ? r : c;
    bytes += 2 * bytes_of(r, c, es) + 2 * bytes_of(s, s, es);
    most = r * c > most ? r * c : most;
    live.push_back(i);
  }
  if (live.empty()) return DTMI_OK;
  size_t thin_ws = 0;
  const NewtonWay way = newton_way(dtype, q, live, thin_ws);
  if (way == kSmall) return run_small(dtype, q, live);
  const int np = norm_blocks(most, es, 512);
  void* ws = nullptr;
  int rc = pool_alloc(&ws, (way == kThin ? thin_ws : bytes) + live.size() * (size_t)np * sizeof(double));
  if (rc) return rc;
  if (way == kThin)
    rc = dtype == DTMI_F32 ? run_thin<float>(dtype, q, live, most, np, (char*)ws)
                           : run_thin<double>(dtype, q, live, most, np, (char*)ws);
  else
    rc = dtype == DTMI_F32 ? newton_run<float>(dtype, q, live, most, np, (char*)ws)
                           : newton_run<double>(dtype, q, live, most, np, (char*)ws);
  pool_free(ws);
  return rc;
}

}  // namespace dtmi

using namespace dtmi;

DTMI_EXPORT int dtmi_newton_schulz(int dtype, int n, void* const* out, const void* const* in, const int64_t* rows,
                                   const int64_t* cols, int steps, double a, double b, double c, double eps) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  NewtonArgs q{};
  q.n = n;
  q.steps = steps;
  q.g = in;
  q.out = out;
  q.rows = rows;
  q.cols = cols;
  q.a = a;
  q.b = b;
  q.c = c;
  q.eps = eps;
  q.gscale = 1.0;
  return newton(__func__, dtype, q);
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_muon(int dtype, int n, void* const* p, const void* const* g, void* const* m, const int64_t* rows,
                          const int64_t* cols, const double* rate, double keep, double momentum, int nesterov,
                          int steps, double a, double b, double c, double eps, double gscale,
                          const double* gscale_dev) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  DTMI_CHECK(n <= 0 || (m && rate), "%s: NULL array", __func__);
  std::vector<double> minus((size_t)(n > 0 ? n : 0));
  for (int i = 0; i < n; ++i) minus[i] = -rate[i];
  NewtonArgs q{};
  q.n = n;
  q.steps = steps;
  q.nesterov = nesterov;
  q.g = g;
  q.m = m;
  q.out = p;
  q.rows = rows;
  q.cols = cols;
  q.a = a;
  q.b = b;
  q.c = c;
  q.eps = eps;
  q.mu = momentum;
  q.gscale = gscale;
  q.gscale_dev = gscale_dev;
  q.gamma = keep;
  q.rate = minus.data();
  return newton(__func__, dtype, q);
  DTMI_BODY_END
}
