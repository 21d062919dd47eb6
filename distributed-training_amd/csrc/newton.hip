// Orthogonalised updates: Newton-Schulz steps on the singular values of a set of
// matrices, and the optimizer step made of them.
//
//   X = U / (|U|_F + eps);  `steps` times: G = X X^T, H = b G + c G G, X = a X + H X
//
// for a matrix of fewer rows than columns; of a taller one the same with X^T X on the
// right. G and H are symmetric: their products run over the tiles on and below the
// diagonal and mirror the rest, so that a step of an m x n matrix (m <= n) costs m^2 n
// + m^3 + 2 m^2 n operations, a third less than three plain products where m = n. All
// matrices of a call share each launch (gemm_group.h), wide and tall ones apart for G.
// Bound: MFMA; small matrices by the 3 steps launches one after the other.
#include <cmath>
#include <utility>
#include <vector>

#include "gemm_group.h"
#include "seqmath.h"

namespace dtmi {

constexpr int kNormParts = 64;   // blocks that share a matrix's sum of squares
constexpr int kNormTasks = 64;   // 40 bytes each: the arguments stay below 4 KB

struct NormTask {
  const void* g;
  void* m;  // momentum (NULL: u = g)
  void* x;  // u / (|u| + eps)
  int64_t n;
  double* part;  // [kNormParts]
};

struct NormArgs {
  int count, nesterov;
  double mu, eps, gscale;
  const double* gscale_dev;
  NormTask t[kNormTasks];
};

// The elements of block `part`: a range of whole vectors, the last block's to the end.
__device__ __forceinline__ void norm_range(int64_t n, int part, int64_t& lo, int64_t& hi) {
  const int64_t per = ((n + kNormParts - 1) / kNormParts + 3) / 4 * 4;
  lo = part * per < n ? part * per : n;
  hi = lo + per < n ? lo + per : n;
}

// PASS 0: m = mu m + g and the block's sum of squares of u = g + mu m (nesterov) or m;
// PASS 1: x = u / (|u| + eps), u formed again from g and m (u itself would be written
// and read once more). Sums in float64. V elements at a time.
template <typename T, int PASS, int V>
__device__ __forceinline__ void norm_body(const NormArgs& a, const NormTask& k, int64_t lo, int64_t hi, T gs, T mu,
                                          double scale, double& sq) {
  const T* __restrict__ G = (const T*)k.g;
  T* __restrict__ M = (T*)k.m;
  T* __restrict__ X = (T*)k.x;
  for (int64_t i = lo + (int64_t)threadIdx.x * V; i + V <= hi; i += 256 * V) {
    T u[V];
    vload<T, V>(u, G + i);
#pragma unroll
    for (int e = 0; e < V; ++e) u[e] = u[e] * gs;
    if (M) {
      T m[V];
      vload<T, V>(m, M + i);
      if constexpr (PASS == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) m[e] = fma(mu, m[e], u[e]);
        vstore<T, V>(M + i, m);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) u[e] = a.nesterov ? fma(mu, m[e], u[e]) : m[e];
    }
    if constexpr (PASS == 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) sq += (double)u[e] * (double)u[e];
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) u[e] = (T)((double)u[e] * scale);
      vstore<T, V>(X + i, u);
    }
  }
}

template <typename T, int PASS>
__global__ void __launch_bounds__(256) norm_kernel(NormArgs a) {
  const NormTask k = a.t[blockIdx.y];
  const T gs = a.gscale_dev ? (T)*a.gscale_dev : (T)a.gscale;
  __shared__ double sh[4];
  double scale = 0.0, sq = 0.0;
  if constexpr (PASS == 1) {
    double s = k.part[threadIdx.x & 63];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    scale = 1.0 / (sqrt(s) + a.eps);
  }
  int64_t lo, hi;
  norm_range(k.n, blockIdx.x, lo, hi);
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec = aligned(k.g, 16) && aligned(k.m, 16) && aligned(k.x, 16);
  const int64_t mid = vec ? lo + (hi - lo) / V * V : lo;
  if (vec) norm_body<T, PASS, V>(a, k, lo, mid, gs, (T)a.mu, scale, sq);
  norm_body<T, PASS, 1>(a, k, mid, hi, gs, (T)a.mu, scale, sq);
  if constexpr (PASS == 0) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sq += __shfl_xor(sq, o, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sq;
    __syncthreads();
    if (threadIdx.x == 0) k.part[blockIdx.x] = (sh[0] + sh[1]) + (sh[2] + sh[3]);
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

template <typename T>
static int newton_run(int dtype, const NewtonArgs& q, const std::vector<int>& live, char* ws, size_t es) {
  const int n = (int)live.size();
  // the workspace: norm parts, then per matrix X twice and G and H
  std::vector<char*> x0(n), x1(n), G(n), H(n);
  double* parts = (double*)ws;
  char* p = ws + (size_t)n * kNormParts * sizeof(double);
  for (int i = 0; i < n; ++i) {
    const int64_t r = q.rows[live[i]], c = q.cols[live[i]], s = r < c ? r : c;
    const size_t xb = ((size_t)r * c * es + 255) & ~(size_t)255, gb = ((size_t)s * s * es + 255) & ~(size_t)255;
    x0[i] = p;
    x1[i] = p + xb;
    G[i] = p + 2 * xb;
    H[i] = G[i] + gb;
    p = H[i] + gb;
  }
  for (int lo = 0; lo < n; lo += kNormTasks) {
    NormArgs a{};
    a.count = n - lo < kNormTasks ? n - lo : kNormTasks;
    a.nesterov = q.nesterov;
    a.mu = q.mu;
    a.eps = q.eps;
    a.gscale = q.gscale;
    a.gscale_dev = q.gscale_dev;
    double bytes = 0;
    for (int i = 0; i < a.count; ++i) {
      const int j = live[lo + i];
      a.t[i] = {q.g[j], q.m ? q.m[j] : nullptr, x0[lo + i], q.rows[j] * q.cols[j], parts + (size_t)(lo + i) * kNormParts};
      bytes += (double)a.t[i].n * (double)es * (q.m ? 6 : 3);
    }
    TimedLaunch tl(DTMI_FAM_OTHER, bytes);
    const dim3 grid(kNormParts, (unsigned)a.count);
    norm_kernel<T, 0><<<grid, 256, 0, stream()>>>(a);
    norm_kernel<T, 1><<<grid, 256, 0, stream()>>>(a);
    LAUNCH_CHECK("norm_kernel");
  }
  std::vector<GroupTask> wide, tall, sq(n), ap(n);
  for (int s = 0; s < q.steps; ++s) {
    const bool last = s + 1 == q.steps;
    wide.clear();
    tall.clear();
    for (int i = 0; i < n; ++i) {
      const int j = live[i], r = (int)q.rows[j], c = (int)q.cols[j], m = r < c ? r : c;
      // G = X X^T, or X^T X of a tall matrix
      (r <= c ? wide : tall).push_back({x0[i], x0[i], G[i], nullptr, m, m, r < c ? c : r, 0, 1.0});
      // H = b G + c G G: G is symmetric, so either operand may be read either way
      sq[i] = {G[i], G[i], H[i], G[i], m, m, m, 0, 1.0};
      // X = a X + H X, or a X + X H; the last into the result
      ap[i] = {r <= c ? H[i] : x0[i], r <= c ? x0[i] : H[i], last ? (char*)q.out[j] : x1[i], x0[i], r, c, m, 0,
               last && q.rate ? q.rate[j] : 1.0};
    }
    int rc = DTMI_OK;
    if (!wide.empty()) rc = run_group(dtype, 1, 1, wide.data(), (int)wide.size(), kDNone, 1, 1.0, 0.0, 0.0);
    if (!rc && !tall.empty()) rc = run_group(dtype, 0, 0, tall.data(), (int)tall.size(), kDNone, 1, 1.0, 0.0, 0.0);
    if (!rc) rc = run_group(dtype, 1, 1, sq.data(), n, kDMatrix, 1, q.c, q.b, 0.0);
    if (!rc) rc = run_group(dtype, 1, 0, ap.data(), n, kDMatrix, 0, 1.0, q.a, last && q.rate ? q.gamma : 0.0);
    if (rc) return rc;
    std::swap(x0, x1);
  }
  return DTMI_OK;
}

static int newton(const char* what, int dtype, const NewtonArgs& q) {
  DTMI_CHECK(q.n >= 0 && q.steps >= 1 && q.steps <= 64, "%s: needs 1 to 64 steps, not %d", what, q.steps);
  DTMI_CHECK(q.n == 0 || (q.g && q.out && q.rows && q.cols), "%s: NULL array", what);
  const size_t es = dtype == DTMI_F32 ? 4 : 8;
  std::vector<int> live;
  size_t bytes = 0;
  for (int i = 0; i < q.n; ++i) {
    const int64_t r = q.rows[i], c = q.cols[i];
    DTMI_CHECK(r >= 0 && c >= 0, "%s: negative size of matrix %d", what, i);
    if (r == 0 || c == 0) continue;
    const int64_t most = (1 << 24) / (int64_t)es;
    DTMI_CHECK(r < most && c < most, "%s: matrix %d, %lld x %lld, has rows or columns of 2^24 bytes or more", what, i,
               (long long)r, (long long)c);
    DTMI_CHECK(q.g[i] && q.out[i] && (!q.m || q.m[i]), "%s: NULL pointer of matrix %d", what, i);
    const int64_t s = r < c ? r : c;
    bytes += (size_t)kNormParts * sizeof(double) + 2 * (((size_t)r * c * es + 255) & ~(size_t)255) +
             2 * (((size_t)s * s * es + 255) & ~(size_t)255);
    live.push_back(i);
  }
  if (live.empty()) return DTMI_OK;
  void* ws = nullptr;
  int rc = pool_alloc(&ws, bytes);
  if (rc) return rc;
  rc = dtype == DTMI_F32 ? newton_run<float>(dtype, q, live, (char*)ws, es)
                         : newton_run<double>(dtype, q, live, (char*)ws, es);
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
