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
// piece. Rows whose target is to be ignored are left out first: see lxent_rows_kernel.
#include <cmath>
#include <vector>

#include "gemm_direct_tile.h"
#include "gemm_group.h"

namespace dtmi {

// Logits of a piece, in bytes: pieces of fewer rows read and write dw more often, 8 C V
// bytes against 6 rows C V operations: 8192 x 768 x 50304 takes 15.1 ms in pieces of 2048
// rows, 14.5 in these (4096).
constexpr int64_t kPieceBytes = 1LL << 30, kPieceRows = 1024;

// Ignored rows are left out where a gradient is asked for (their x may hold anything, and
// 0 x NaN would reach dw) or where their products are more operations than this, 16 us in
// float32: leaving them out is three more launches (8 rows of 1039 words: 24 us a call in
// place, 54 us when the host made the list).
constexpr double kLeaveOut = 2e9;

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

// The rows whose target is not `ignore`, in order: sel their numbers, t their targets, and
// for every row its place among them or -1. One block, four rows a thread at a time
// (2683 rows: 3.4 us). n is the caller's count: no more are written, and what a count too
// large leaves over names row 0.
__global__ void __launch_bounds__(1024) lxent_rows_kernel(const int64_t* __restrict__ targets, int64_t R,
                                                          int64_t ignore, int64_t n, int* __restrict__ sel,
                                                          int64_t* __restrict__ t, int* __restrict__ place) {
  constexpr int U = 4;
  __shared__ int sh[2][U][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t base = 0;
  for (int64_t r0 = 0, turn = 0; r0 < R; r0 += 1024 * U, turn ^= 1) {
    int64_t v[U];
    uint64_t in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * 1024 + threadIdx.x;
      v[u] = r < R ? targets[r] : ignore;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      in[u] = __ballot(v[u] != ignore);
      if (lane == 0) sh[turn][u][wave] = __popcll(in[u]);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * 1024 + threadIdx.x;
      int before = 0, total = 0;
      for (int w = 0; w < 16; ++w) {
        const int c = sh[turn][u][w];
        before += w < wave ? c : 0;
        total += c;
      }
      const int64_t at = base + before + __popcll(in[u] & ((1ULL << lane) - 1));
      const bool kept = v[u] != ignore && at < n;
      if (r < R) place[r] = kept ? (int)at : -1;
      if (kept) {
        sel[at] = (int)r;
        t[at] = v[u];
      }
      base += total;
    }
  }
  for (int64_t i = base + threadIdx.x; i < n; i += 1024) {
    sel[i] = 0;
    t[i] = 0;
  }
}

// out row r = in row from[r], 0 where that is negative; lanes threads a row.
template <typename T>
__global__ void __launch_bounds__(256) lxent_pick_kernel(T* __restrict__ out, const T* __restrict__ in,
                                                         const int* __restrict__ from, int64_t rows, int64_t cols,
                                                         int lanes) {
  const int64_t r = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  if (r >= rows) return;
  const int64_t f = from[r];
  for (int64_t c = threadIdx.x % lanes; c < cols; c += lanes) out[r * cols + c] = f >= 0 ? in[f * cols + c] : T(0);
}

template <typename T>
static int pick_rows(T* out, const T* in, const int* from, int64_t rows, int64_t cols) {
  if (!rows || !cols) return DTMI_OK;
  const int lanes = cols >= 32 ? 64 : 1;
  TimedLaunch tl(DTMI_FAM_OTHER, 2.0 * (double)(rows * cols) * (double)sizeof(T));
  lxent_pick_kernel<T><<<(unsigned)cdiv(rows, 256 / lanes), 256, 0, stream()>>>(out, in, from, rows, cols, lanes);
  LAUNCH_CHECK("lxent_pick_kernel");
  return DTMI_OK;
}

// A row's statistics from its parts, joined in a fixed order: ROWS rows a block, on
// consecutive lanes, the parts dealt to 1024 / ROWS groups that are joined through LDS.
// 32 rows read whole lines of the parts; with few rows one a block is quicker, as no lane
// then walks more than a few parts (5 rows of 1572 parts: 9 us with 32 rows a block).
template <typename T, int ROWS>
__global__ void __launch_bounds__(1024) lxent_join_kernel(const T* __restrict__ pmax, const T* __restrict__ psum,
                                                          int64_t parts, int64_t M, const T* __restrict__ zt,
                                                          const int64_t* __restrict__ targets, int64_t ignore,
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
    rmax[m] = x.m;
    rsum[m] = x.s;
    // log(sum) + (max - z): the difference first, as both may be large
    losses[m] = targets[m] == ignore ? T(0) : log(x.s) + (x.m - zt[m]);
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

// The join and the mean together, for as few rows and parts as one block goes through at
// once: a thread a row.
constexpr int64_t kJoinMeanRows = 1024, kJoinMeanParts = 16;
template <typename T>
__global__ void __launch_bounds__(1024) lxent_join_mean_kernel(const T* __restrict__ pmax, const T* __restrict__ psum,
                                                               int parts, int M, const T* __restrict__ zt,
                                                               const int64_t* __restrict__ targets, int64_t ignore,
                                                               T* __restrict__ rmax, T* __restrict__ rsum,
                                                               T* __restrict__ losses, double coef,
                                                               T* __restrict__ mean) {
  __shared__ double sh[16];
  const int m = threadIdx.x;
  double l = 0.0;
  if (m < M) {
    RowStat<T> x;
    for (int p = 0; p < parts; ++p) x.add(pmax[(int64_t)p * M + m], psum[(int64_t)p * M + m]);
    const T loss = targets[m] == ignore ? T(0) : log(x.s) + (x.m - zt[m]);
    rmax[m] = x.m;
    rsum[m] = x.s;
    losses[m] = loss;
    l = (double)loss;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o, 64);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = l;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0.0;
    for (int i = 0; i < 16; ++i) t += sh[i];
    *mean = (T)(t * coef);
  }
}

// dz in place of z: block (x, y) takes 4 vectors a thread of rows y, y + gridDim.y, ...
// Vectors need element alignment only, so a vocabulary that is no multiple of one runs the
// same, with its last few elements one by one (1067 x 50257: 104 us element by element).
// sel: the rows' own numbers, which g goes by, where some were left out.
template <typename T>
__global__ void __launch_bounds__(256) lxent_dz_kernel(T* __restrict__ z, int64_t rows, int64_t cols,
                                                       const T* __restrict__ rmax, const T* __restrict__ rsum,
                                                       const int64_t* __restrict__ targets, const int* __restrict__ sel,
                                                       const T* __restrict__ g, int64_t g_stride, double coef) {
  constexpr int V = 16 / (int)sizeof(T);
  typedef typename UVec<T>::type vt;
  const int64_t c0 = (int64_t)blockIdx.x * (256 * 4 * V);
  for (int64_t m = blockIdx.y; m < rows; m += gridDim.y) {
    T* row = z + m * cols;
    const T mx = rmax[m], c = g ? (T)coef * g[(sel ? sel[m] : m) * g_stride] : (T)coef;
    const T inv = T(1) / rsum[m];
    const int64_t t = targets[m];
    auto dz = [&](T x, int64_t at) {
      const T p = exp_e<T>(x - mx) * inv;
      return c * (at == t ? p - T(1) : p);
    };
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = c0 + (u * 256 + threadIdx.x) * V;
      if (at + V <= cols) {
        typename MF<T>::vec_t v = *reinterpret_cast<const vt*>(row + at);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = dz(v[e], at + e);
        *reinterpret_cast<vt*>(row + at) = v;
      } else {
        for (int64_t i = at; i < cols; ++i) row[i] = dz(row[i], i);
      }
    }
  }
}

struct LxentArgs {
  int64_t R, C, V;
  const char *X, *W;
  int tied;
  const void* b;
  const int64_t* targets;
  int64_t counted, ignore;
  char* losses;
  void* mean;
  const char* g;
  int64_t g_stride;
  double coef;
  char *dX, *dW, *db;
  const int* sel = nullptr;  // the rows' numbers, where some are left out
};

// Pool memory that goes back at the end of the call's enqueuing.
struct Scratch {
  void* p = nullptr;
  ~Scratch() {
    if (p) pool_free(p);
  }
};

// Whether the products run in the type they are in: the split bf16 arithmetic is the GEMM's.
template <typename T>
static bool plain_products() {
  int math = DTMI_GEMM_MATH_F32;
  return sizeof(T) == 8 || (dtmi_get_gemm_math(&math) == DTMI_OK && math == DTMI_GEMM_MATH_F32);
}

// Whether a piece's gradients are products of gemm_group.h, whose ragged last rounds cost
// less than the GEMM's: the largest (4096 x 768 x 50304, dw 2.13 ms and 2.32, dx 2.18 and
// 2.18), and odd sizes (1067 x 515 x 50257 517 and 546 us, 531 and 565; float64 1000 x 385 x
// 8001 123 and 145, 132 and 158). Others are quicker by the GEMM (4000 x 384 x 8000, dw 194
// and 213 us).
template <typename T>
static bool grouped(int64_t R, int64_t C, int64_t V) {
  if (!plain_products<T>()) return false;
  const double operations = 2.0 * (double)R * (double)C * (double)V;
  return operations >= 1e11 || (operations >= 1e9 && (C % MF<T>::VEC || V % MF<T>::VEC));
}

// dx of few rows: their products split the vocabulary over more blocks than the GEMM's tiles
// do (8 x 175 x 26217 15 us and 53, 32 x 515 x 50257 57 and 93, 4 x 605 x 1055 13 and 9).
constexpr int64_t kFewRows = 32, kFewWords = 2000;

// dw, db and dx of a piece of n rows with its dz in Z. dx last: it may take x's place.
template <typename T>
static int grad_products(int dtype, const LxentArgs& q, int64_t n, char* Z, const char* X, char* dX, int add) {
  const int rows = (int)n, C = (int)q.C, V = (int)q.V;
  const bool group = grouped<T>(n, q.C, q.V);
  int rc = DTMI_OK;
  if (group) {
    const bool sums = q.db && q.dW && !q.tied;  // db by the tiles of dw
    std::vector<GroupLaunch> l;
    if (q.dW) {
      const GroupTask t = q.tied ? GroupTask{Z, X, q.dW, nullptr, V, C, rows, 0, 1.0}
                                 : GroupTask{X, Z, q.dW, sums ? q.db : nullptr, C, V, rows, 0, 1.0};
      rc = plan_group(dtype, 0, 0, {t}, sums ? kDColsum : kDNone, 0, 1.0, 0.0, add ? 1.0 : 0.0, 1, 1, l);
      if (!rc) rc = launch_group(dtype, l);
    }
    if (!rc && q.db && !sums) rc = dtmi_colsum(dtype, q.db, Z, n, q.V, add);
  } else if (q.tied) {
    if (q.dW) rc = dtmi_gemm(dtype, 0, 0, q.V, q.C, n, Z, q.V, 0, X, q.C, 0, q.dW, q.C, 0, 1, nullptr, add, 0);
    if (!rc && q.db) rc = dtmi_colsum(dtype, q.db, Z, n, q.V, add);
  } else if (q.dW) {
    rc = dtmi_linear_bwd_dw(dtype, q.dW, q.db, X, Z, n, q.C, q.V, add);
  } else if (q.db) {
    rc = dtmi_colsum(dtype, q.db, Z, n, q.V, add);
  }
  if (rc || !dX || C == 0) return rc;
  if (group || (n <= kFewRows && V >= kFewWords && plain_products<T>())) {
    std::vector<GroupLaunch> l;
    rc = plan_group(dtype, 1, q.tied ? 0 : 1, {GroupTask{Z, q.W, dX, nullptr, rows, C, V, 0, 1.0}}, kDNone, 0, 1.0, 0.0,
                    0.0, 1, 1, l);
    return rc ? rc : launch_group(dtype, l);
  }
  return q.tied ? dtmi_gemm(dtype, 1, 0, n, q.C, q.V, Z, q.V, 0, q.W, q.C, 0, dX, q.C, 0, 1, nullptr, 0, 0)
                : dtmi_linear_bwd_dx(dtype, dX, Z, q.W, n, q.C, q.V, 0);
}

template <typename T>
static int lxent_pieces(int dtype, const LxentArgs& q, int64_t piece, char* Z, char* stats) {
  constexpr int64_t es = sizeof(T);
  const bool grads = q.dX || q.dW || q.db;
  bool joint = false;
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
    int rc = run_stats(dtype, q.tied, a);
    if (rc) return rc;
    joint = q.mean && n == q.R && n <= kJoinMeanRows && parts <= kJoinMeanParts;
    {
      TimedLaunch tl(DTMI_FAM_XENT, 2.0 * (double)(parts * n) * es);
      if (joint)
        lxent_join_mean_kernel<T><<<1, 1024, 0, stream()>>>(pmax, psum, (int)parts, (int)n, zt, a.targets, q.ignore,
                                                            rmax, rsum, losses, q.coef, (T*)q.mean);
      else if (n <= 512)
        lxent_join_kernel<T, 1><<<(unsigned)n, 1024, 0, stream()>>>(pmax, psum, parts, n, zt, a.targets, q.ignore, rmax,
                                                                    rsum, losses);
      else
        lxent_join_kernel<T, 32><<<(unsigned)cdiv(n, 32), 1024, 0, stream()>>>(pmax, psum, parts, n, zt, a.targets,
                                                                               q.ignore, rmax, rsum, losses);
    }
    if (grads) {
      {
        TimedLaunch tl(DTMI_FAM_XENT, 2.0 * (double)n * (double)q.V * es);
        constexpr int V = 16 / (int)sizeof(T);
        const T* g = (const T*)q.g + (q.g && !q.sel ? lo * q.g_stride : 0);
        const unsigned ny = (unsigned)(n < 32768 ? n : 32768);
        lxent_dz_kernel<T><<<dim3((unsigned)cdiv(q.V, 1024 * V), ny), 256, 0, stream()>>>(
            (T*)Z, n, q.V, rmax, rsum, a.targets, q.sel ? q.sel + lo : nullptr, g, q.g_stride, q.coef);
      }
      LAUNCH_CHECK("lxent_dz_kernel");
      rc = grad_products<T>(dtype, q, n, Z, X, q.dX ? q.dX + lo * q.C * es : nullptr, lo > 0);
      if (rc) return rc;
    }
    LAUNCH_CHECK("lxent kernels");
  }
  if (q.mean && !joint) {
    lxent_mean_kernel<T><<<1, 1024, 0, stream()>>>((const T*)q.losses, q.R, q.coef, (T*)q.mean);
    LAUNCH_CHECK("lxent_mean_kernel");
  }
  return DTMI_OK;
}

template <typename T>
static int lxent_counted(int dtype, LxentArgs q) {
  constexpr int64_t es = sizeof(T);
  const bool grads = q.dX || q.dW || q.db;
  Scratch losses, Z, stats;
  int rc = DTMI_OK;
  if (!q.losses) {
    rc = pool_alloc(&losses.p, (size_t)(q.R * es));
    if (rc) return rc;
    q.losses = (char*)losses.p;
  }
  int64_t piece = q.R;
  if (grads) {
    int64_t most = kPieceBytes / (q.V * es);
    most = most < kPieceRows ? kPieceRows : most;
    piece = cdiv(cdiv(q.R, cdiv(q.R, most)), 128) * 128;
    if (piece > q.R) piece = q.R;
    rc = pool_alloc(&Z.p, (size_t)(piece * q.V * es));
    while (rc == DTMI_ERR_OOM && piece > 128) {  // smaller pieces where memory is short
      piece = cdiv(piece / 2, 128) * 128;
      rc = pool_alloc(&Z.p, (size_t)(piece * q.V * es));
    }
    if (rc) return rc;
  }
  const int64_t tail = q.R % piece;
  int64_t parts = stats_parts(dtype, q.tied, piece, q.V, q.C);
  if (tail) {
    const int64_t p = stats_parts(dtype, q.tied, tail, q.V, q.C);
    parts = p > parts ? p : parts;
  }
  rc = pool_alloc(&stats.p, (size_t)((3 + 2 * parts) * piece * es));
  return rc ? rc : lxent_pieces<T>(dtype, q, piece, (char*)Z.p, (char*)stats.p);
}

// The rows that count, by themselves: their x, or where a gradient of it is asked for the
// gradient in its place, in a workspace.
template <typename T>
static int lxent_run(int dtype, const LxentArgs& q) {
  constexpr int64_t es = sizeof(T);
  const bool grads = q.dX || q.dW || q.db;
  const int64_t n = q.counted;
  if (n == q.R || (!grads && 2.0 * (double)(q.R - n) * (double)q.C * (double)q.V < kLeaveOut))
    return lxent_counted<T>(dtype, q);
  Scratch rows, x;
  int rc = pool_alloc(&rows.p, (size_t)(n * 8 + (n + q.R) * 4 + n * es + 8));
  if (!rc) rc = pool_alloc(&x.p, (size_t)(n * q.C * es + 8));
  if (rc) return rc;
  int64_t* t = (int64_t*)rows.p;
  T* ls = (T*)(t + n);
  int* sel = (int*)(ls + n);
  int* place = sel + n;
  {
    TimedLaunch tl(DTMI_FAM_OTHER, (double)(q.R + n) * 12.0);
    lxent_rows_kernel<<<1, 1024, 0, stream()>>>(q.targets, q.R, q.ignore, n, sel, t, place);
  }
  LAUNCH_CHECK("lxent_rows_kernel");
  rc = pick_rows((T*)x.p, (const T*)q.X, sel, n, q.C);
  if (rc) return rc;
  LxentArgs c = q;
  c.R = n;
  c.X = (const char*)x.p;
  c.targets = t;
  c.losses = (char*)ls;
  if (q.dX) c.dX = (char*)x.p;
  c.sel = sel;
  rc = lxent_counted<T>(dtype, c);
  if (!rc && q.dX) rc = pick_rows((T*)q.dX, (const T*)x.p, place, q.R, q.C);
  if (!rc && q.losses) rc = pick_rows((T*)q.losses, ls, place, q.R, 1);
  return rc;
}

struct ScaleArgs {
  void* p[3];
  int64_t n[3];
};

// blockIdx.y: the array. Leaves at once for a factor of 1.
template <typename T>
__global__ void __launch_bounds__(256) grad_scale_kernel(ScaleArgs a, const T* __restrict__ g) {
  const T f = g[0];
  if (f == T(1)) return;
  constexpr int V = 16 / (int)sizeof(T);
  typedef T vt __attribute__((ext_vector_type(V)));
  T* p = (T*)a.p[blockIdx.y];
  const int64_t n = a.n[blockIdx.y], nv = aligned(p, 16) ? n / V : 0, stride = (int64_t)gridDim.x * 256;
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = i0; i < nv; i += stride) reinterpret_cast<vt*>(p)[i] *= f;
  for (int64_t i = nv * V + i0; i < n; i += stride) p[i] *= f;
}

}  // namespace dtmi

using namespace dtmi;

DTMI_EXPORT int dtmi_linear_xent(int dtype, int64_t R, int64_t C, int64_t V, const void* X, const void* W, int tied,
                                 const void* b, const int64_t* targets, int64_t counted, int64_t ignore, void* losses,
                                 void* mean, const void* g, int64_t g_stride, double coef, void* dX, void* dW,
                                 void* db) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  DTMI_CHECK(R >= 0 && C >= 0 && V >= 1, "%s: bad sizes R=%lld C=%lld V=%lld", __func__, (long long)R, (long long)C,
             (long long)V);
  DTMI_CHECK(R < (1LL << 31) && C < (1LL << 22) && V < (1LL << 22), "%s: too large", __func__);
  DTMI_CHECK(g_stride == 0 || g_stride == 1, "%s: g_stride must be 0 or 1", __func__);
  DTMI_CHECK(counted >= 0 && counted <= R, "%s: %lld of %lld rows that count", __func__, (long long)counted,
             (long long)R);
  if (counted == 0) {
    int rc = mean ? dtmi_fill(dtype, mean, 0.0, 1) : DTMI_OK;
    if (!rc && dW) rc = dtmi_fill(dtype, dW, 0.0, C * V);
    if (!rc && db) rc = dtmi_fill(dtype, db, 0.0, V);
    if (!rc && dX) rc = dtmi_fill(dtype, dX, 0.0, R * C);
    if (!rc && losses) rc = dtmi_fill(dtype, losses, 0.0, R);
    return rc;
  }
  DTMI_CHECK(targets && (C == 0 || (X && W)), "%s: NULL pointer", __func__);
  LxentArgs q{R, C, V, (const char*)X, (const char*)W, tied ? 1 : 0, b, targets, counted,
              counted < R ? ignore : INT64_MIN, (char*)losses, mean, (const char*)g, g_stride, coef,
              (char*)dX, (char*)dW, (char*)db};
  return dtype == DTMI_F32 ? lxent_run<float>(dtype, q) : lxent_run<double>(dtype, q);
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_grad_scale_multi(int dtype, int n, void* const* ptrs, const int64_t* counts, const void* g_dev) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  DTMI_CHECK(n >= 1 && n <= 3 && ptrs && counts && g_dev, "%s: 1 to 3 arrays and a factor", __func__);
  ScaleArgs a{};
  int64_t most = 0, total = 0;
  for (int i = 0; i < n; ++i) {
    DTMI_CHECK(counts[i] >= 0 && (counts[i] == 0 || ptrs[i]), "%s: bad array %d", __func__, i);
    a.p[i] = ptrs[i];
    a.n[i] = counts[i];
    most = counts[i] > most ? counts[i] : most;
    total += counts[i];
  }
  if (!most) return DTMI_OK;
  TimedLaunch tl(DTMI_FAM_OTHER, 2.0 * (double)total * (dtype == DTMI_F32 ? 4 : 8));
  const int64_t blocks = cdiv(most, 4096);
  const dim3 grid((unsigned)(blocks < 2048 ? blocks : 2048), (unsigned)n);
  if (dtype == DTMI_F32)
    grad_scale_kernel<float><<<grid, 256, 0, stream()>>>(a, (const float*)g_dev);
  else
    grad_scale_kernel<double><<<grid, 256, 0, stream()>>>(a, (const double*)g_dev);
  LAUNCH_CHECK("grad_scale_kernel");
  return DTMI_OK;
  DTMI_BODY_END
}
