// Softmax cross entropy of x w + b over a large vocabulary without the logits: the
// losses from row statistics that the product's own epilogue takes (no logits at
// all), the gradients over pieces of the rows, whose logits live in one workspace.
//
//   l_r = log sum_v exp z_rv - z_r,t(r);  dz_rv = c_r (exp z_rv / sum - [v = t(r)])
//   dx = dz w^T, dw = x^T dz, db = sum_r dz
//
// Bound: MFMA, 2 R C V operations for the losses and 6 R C V with gradients; up to
// about 30 rows reading w. A gradient needs a row's whole sum before its first element,
// so pieces of the vocabulary would form every logit twice (8 R C V); pieces of the
// rows form them once, and add up dw over them, which costs one read and write of it a
// piece.
#include <cmath>

#include "gemm_group.h"

namespace dtmi {

// Rows of a piece. Fewer rows read and write dw more often, 8 C V bytes against 6 rows
// C V operations; more take rows * V * 4 bytes of workspace.
constexpr int64_t kPieceRows = 2048;

template <typename T>
__device__ __forceinline__ T exp_e(T x) {
  if constexpr (sizeof(T) == 4) return __builtin_amdgcn_exp2f(x * 1.44269504f);
  return exp(x);
}

template <typename T>
struct RowStat {
  T m = -INFINITY, s = T(0);
  // NaN: dropped by the maximum, kept by the sum; parts of -inf alone have sum 0
  __device__ __forceinline__ void add(T m2, T s2) {
    const T top = fmax(m, m2), ref = top == -INFINITY ? T(0) : top;
    s = s * exp_e<T>(m - ref) + s2 * exp_e<T>(m2 - ref);
    m = top;
  }
};

// A row's statistics from its parts, joined in a fixed order: ROWS rows a block, on
// consecutive lanes, the parts dealt to 1024 / ROWS groups that are joined through LDS.
// 32 rows read whole lines of the parts; with few rows one a block is quicker, as no lane
// then walks more than a few parts (5 rows of 1572 parts: 9 us with 32 rows a block).
template <typename T, int ROWS>
__global__ void __launch_bounds__(1024) lxent_join_kernel(const T* __restrict__ pmax, const T* __restrict__ psum,
                                                          int64_t parts, int64_t M, const T* __restrict__ zt,
                                                          T* __restrict__ rmax, T* __restrict__ rsum,
                                                          T* __restrict__ losses) {
  constexpr int GROUPS = 1024 / ROWS, U = ROWS == 1 ? 2 : 8;
  __shared__ T sm[GROUPS][ROWS + 1], ss[GROUPS][ROWS + 1];
  const int r = threadIdx.x % ROWS, grp = threadIdx.x / ROWS;
  const int64_t m = (int64_t)blockIdx.x * ROWS + r;
  RowStat<T> x;
  if (m < M) {
    for (int64_t p0 = grp; p0 < parts; p0 += GROUPS * U) {
      T a[U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t p = p0 + GROUPS * u;
        const int64_t at = (p < parts ? p : p0) * M + m;
        a[u] = pmax[at];
        b[u] = p < parts ? psum[at] : T(0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) x.add(a[u], b[u]);
    }
  }
  sm[grp][r] = x.m;
  ss[grp][r] = x.s;
  __syncthreads();
#pragma unroll
  for (int half = GROUPS / 2; half >= 1; half >>= 1) {
    if (grp < half) {
      x.add(sm[grp + half][r], ss[grp + half][r]);
      sm[grp][r] = x.m;
      ss[grp][r] = x.s;
    }
    __syncthreads();
  }
  if (grp == 0 && m < M) {
    if (rmax) {
      rmax[m] = x.m;
      rsum[m] = x.s;
    }
    // log(sum) + (max - z): the difference first, as both may be large
    if (losses) losses[m] = log(x.s) + (x.m - zt[m]);
  }
}

// mean = coef * sum of the losses, in float64 and in a fixed order: one block.
template <typename T>
__global__ void __launch_bounds__(1024) lxent_mean_kernel(const T* __restrict__ losses, int64_t n, double coef,
                                                          T* __restrict__ mean) {
  __shared__ double sh[16];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += (double)losses[i];
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < 16; ++i) t += sh[i];
    *mean = (T)(t * coef);
  }
}

// dz in place of z: block (x, y) takes 4 vectors a thread of row y.
template <typename T, int V>
__global__ void __launch_bounds__(256) lxent_dz_kernel(T* __restrict__ z, int64_t cols, const T* __restrict__ rmax,
                                                       const T* __restrict__ rsum, const int64_t* __restrict__ targets,
                                                       const T* __restrict__ g, int64_t g_stride, double coef) {
  typedef T vt __attribute__((ext_vector_type(V == 1 ? 2 : V)));
  const int64_t m = blockIdx.y;
  T* row = z + m * cols;
  const T mx = rmax[m], c = g ? (T)coef * g[m * g_stride] : (T)coef;
  const T inv = T(1) / rsum[m];
  const int64_t t = targets[m];
  const int64_t c0 = (int64_t)blockIdx.x * (256 * 4 * V);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t at = c0 + (u * 256 + threadIdx.x) * V;
    if (at >= cols) continue;
    if constexpr (V == 1) {
      const T p = exp_e<T>(row[at] - mx) * inv;
      row[at] = c * (at == t ? p - T(1) : p);
    } else {
      vt v = *reinterpret_cast<const vt*>(row + at);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const T p = exp_e<T>(v[e] - mx) * inv;
        v[e] = c * (at + e == t ? p - T(1) : p);
      }
      *reinterpret_cast<vt*>(row + at) = v;
    }
  }
}

struct LxentArgs {
  int64_t R, C, V;
  const char *X, *W;
  int tied;
  const void* b;
  const int64_t* targets;
  char* losses;
  void* mean;
  const char* g;
  int64_t g_stride;
  double coef;
  char *dX, *dW, *db;
};

template <typename T>
static int lxent_pieces(int dtype, const LxentArgs& q, int64_t piece, char* Z, char* stats) {
  constexpr int64_t es = sizeof(T);
  const bool grads = q.dX || q.dW || q.db;
  for (int64_t lo = 0; lo < q.R; lo += piece) {
    const int64_t n = q.R - lo < piece ? q.R - lo : piece;
    const int64_t parts = stats_parts(dtype, q.tied, n, q.V, q.C);
    T* rmax = (T*)stats;
    T* rsum = rmax + n;
    T* zt = rsum + n;
    T* pmax = zt + n;
    T* psum = pmax + parts * n;
    const char* X = q.X + lo * q.C * es;
    T* losses = (T*)(q.losses + lo * es);
    StatsArgs a{};
    a.A = X;
    a.B = q.W;
    a.bias = q.b;
    a.C = Z;
    a.pmax = pmax;
    a.psum = psum;
    a.zt = zt;
    a.targets = q.targets + lo;
    a.M = n;
    a.N = q.V;
    a.K = q.C;
    a.lda = q.C;
    a.ldb = q.tied ? q.C : q.V;
    a.ldc = q.V;
    a.nz = q.V;
    int rc = run_stats(dtype, q.tied, a);
    if (rc) return rc;
    {
      TimedLaunch tl(DTMI_FAM_XENT, 2.0 * (double)(parts * n) * es);
      if (n <= 512)
        lxent_join_kernel<T, 1><<<(unsigned)n, 1024, 0, stream()>>>(pmax, psum, parts, n, zt, rmax, rsum, losses);
      else
        lxent_join_kernel<T, 32><<<(unsigned)cdiv(n, 32), 1024, 0, stream()>>>(pmax, psum, parts, n, zt, rmax, rsum,
                                                                               losses);
    }
    if (grads) {
      {
        TimedLaunch tl(DTMI_FAM_XENT, 2.0 * (double)n * (double)q.V * es);
        constexpr int V = 16 / (int)sizeof(T);
        const T* g = q.g ? (const T*)q.g + lo * q.g_stride : nullptr;
        if (q.V % V == 0)
          lxent_dz_kernel<T, V><<<dim3((unsigned)cdiv(q.V, 1024 * V), (unsigned)n), 256, 0, stream()>>>(
              (T*)Z, q.V, rmax, rsum, a.targets, g, q.g_stride, q.coef);
        else
          lxent_dz_kernel<T, 1><<<dim3((unsigned)cdiv(q.V, 1024), (unsigned)n), 256, 0, stream()>>>(
              (T*)Z, q.V, rmax, rsum, a.targets, g, q.g_stride, q.coef);
      }
      LAUNCH_CHECK("lxent_dz_kernel");
      const int add = lo > 0;
      if (q.dX) {
        char* dX = q.dX + lo * q.C * es;
        rc = q.tied ? dtmi_gemm(dtype, 1, 0, n, q.C, q.V, Z, q.V, 0, q.W, q.C, 0, dX, q.C, 0, 1, nullptr, 0, 0)
                    : dtmi_linear_bwd_dx(dtype, dX, Z, q.W, n, q.C, q.V, 0);
        if (rc) return rc;
      }
      if (q.tied) {
        if (q.dW) rc = dtmi_gemm(dtype, 0, 0, q.V, q.C, n, Z, q.V, 0, X, q.C, 0, q.dW, q.C, 0, 1, nullptr, add, 0);
        if (!rc && q.db) rc = dtmi_colsum(dtype, q.db, Z, n, q.V, add);
      } else if (q.dW) {
        rc = dtmi_linear_bwd_dw(dtype, q.dW, q.db, X, Z, n, q.C, q.V, add);
      } else if (q.db) {
        rc = dtmi_colsum(dtype, q.db, Z, n, q.V, add);
      }
      if (rc) return rc;
    }
    LAUNCH_CHECK("lxent kernels");
  }
  if (q.mean) {
    lxent_mean_kernel<T><<<1, 1024, 0, stream()>>>((const T*)q.losses, q.R, q.coef, (T*)q.mean);
    LAUNCH_CHECK("lxent_mean_kernel");
  }
  return DTMI_OK;
}

static int lxent_run(int dtype, LxentArgs& q) {
  const size_t es = dtype == DTMI_F32 ? 4 : 8;
  const bool grads = q.dX || q.dW || q.db;
  void *own = nullptr, *Z = nullptr, *stats = nullptr;
  int64_t piece = q.R;
  int rc = DTMI_OK;
  if (!q.losses) {
    rc = pool_alloc(&own, (size_t)q.R * es);
    if (rc) return rc;
    q.losses = (char*)own;
  }
  if (grads) {
    piece = cdiv(cdiv(q.R, cdiv(q.R, kPieceRows)), 128) * 128;
    if (piece > q.R) piece = q.R;
    rc = pool_alloc(&Z, (size_t)piece * q.V * es);
    while (rc == DTMI_ERR_OOM && piece > 128) {  // smaller pieces where memory is short
      piece = cdiv(piece / 2, 128) * 128;
      rc = pool_alloc(&Z, (size_t)piece * q.V * es);
    }
  }
  if (!rc) {
    const int64_t tail = q.R % piece;
    int64_t parts = stats_parts(dtype, q.tied, piece, q.V, q.C);
    if (tail) {
      const int64_t p = stats_parts(dtype, q.tied, tail, q.V, q.C);
      parts = p > parts ? p : parts;
    }
    rc = pool_alloc(&stats, (size_t)(3 + 2 * parts) * piece * es);
  }
  if (!rc)
    rc = dtype == DTMI_F32 ? lxent_pieces<float>(dtype, q, piece, (char*)Z, (char*)stats)
                           : lxent_pieces<double>(dtype, q, piece, (char*)Z, (char*)stats);
  if (stats) pool_free(stats);
  if (Z) pool_free(Z);
  if (own) pool_free(own);
  return rc;
}

// out row rows[i] = in row i; one wave a row.
template <typename T>
__global__ void __launch_bounds__(256) scatter_rows_kernel(T* __restrict__ out, const T* __restrict__ in,
                                                           const int64_t* __restrict__ rows, int64_t n, int64_t total,
                                                           int64_t cols) {
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (i >= n) return;
  const int64_t r = rows[i];
  if (r < 0 || r >= total) return;
  for (int64_t c = threadIdx.x & 63; c < cols; c += 64) out[r * cols + c] = in[i * cols + c];
}

}  // namespace dtmi

using namespace dtmi;

DTMI_EXPORT int dtmi_linear_xent(int dtype, int64_t R, int64_t C, int64_t V, const void* X, const void* W, int tied,
                                 const void* b, const int64_t* targets, void* losses, void* mean, const void* g,
                                 int64_t g_stride, double coef, void* dX, void* dW, void* db) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  DTMI_CHECK(R >= 0 && C >= 0 && V >= 1, "%s: bad sizes R=%lld C=%lld V=%lld", __func__, (long long)R, (long long)C,
             (long long)V);
  DTMI_CHECK(R < (1LL << 31) && C < (1LL << 22) && V < (1LL << 22), "%s: too large", __func__);
  DTMI_CHECK(g_stride == 0 || g_stride == 1, "%s: g_stride must be 0 or 1", __func__);
  if (R == 0) {
    int rc = mean ? dtmi_fill(dtype, mean, 0.0, 1) : DTMI_OK;
    if (!rc && dW) rc = dtmi_fill(dtype, dW, 0.0, C * V);
    if (!rc && db) rc = dtmi_fill(dtype, db, 0.0, V);
    return rc;
  }
  DTMI_CHECK(targets && (C == 0 || (X && W)), "%s: NULL pointer", __func__);
  LxentArgs q{R, C, V, (const char*)X, (const char*)W, tied ? 1 : 0, b, targets, (char*)losses, mean, (const char*)g,
              g_stride, coef, (char*)dX, (char*)dW, (char*)db};
  return lxent_run(dtype, q);
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_scatter_rows(int dtype, void* out, const void* in, const int64_t* rows, int64_t n, int64_t total,
                                  int64_t cols) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  DTMI_CHECK(n >= 0 && total >= 0 && cols >= 0 && n < (1LL << 31), "%s: bad sizes", __func__);
  if (total == 0 || cols == 0) return DTMI_OK;
  DTMI_CHECK(out && (n == 0 || (in && rows)), "%s: NULL pointer", __func__);
  int rc = dtmi_fill(dtype, out, 0.0, total * cols);
  if (rc || n == 0) return rc;
  TimedLaunch tl(DTMI_FAM_OTHER, 2.0 * (double)(n * cols) * (dtype == DTMI_F32 ? 4 : 8));
  if (dtype == DTMI_F32)
    scatter_rows_kernel<float><<<(unsigned)cdiv(n, 4), 256, 0, stream()>>>((float*)out, (const float*)in, rows, n, total,
                                                                           cols);
  else
    scatter_rows_kernel<double><<<(unsigned)cdiv(n, 4), 256, 0, stream()>>>((double*)out, (const double*)in, rows, n,
                                                                            total, cols);
  LAUNCH_CHECK("scatter_rows_kernel");
  return DTMI_OK;
  DTMI_BODY_END
}
