// Products of experts with ragged sizes: rows off[e] .. off[e + 1] of x [R, K] belong
// to expert e, y = x w[e] + b[e]; dx = g w[e]^T, dw[e] = x^T g, db[e] = the column
// sums of g over the expert's rows. A group of products (gemm_group.h) whose tasks
// are the experts: all of them share one launch, whatever rows each was given.
//
// Bound: MFMA from about 30 rows an expert on (2 R K N operations over E K N
// weights), below that reading the weights of the experts that have rows.
#include <utility>
#include <vector>

#include "gemm_group.h"

namespace dtmi {

// Offsets off[0 .. E] on the host, checked.
static int expert_offsets(const char* what, const int64_t* sizes, int64_t E, int64_t R, int64_t K, int64_t N,
                          std::vector<int64_t>& off) {
  DTMI_CHECK(E >= 0 && R >= 0 && K >= 0 && N >= 0, "%s: negative size", what);
  DTMI_CHECK(R < (1LL << 31) && K < (1LL << 31) && N < (1LL << 31) && E < (1LL << 24), "%s: too large", what);
  DTMI_CHECK(E == 0 || sizes, "%s: NULL sizes", what);
  off.resize((size_t)E + 1);
  off[0] = 0;
  for (int64_t e = 0; e < E; ++e) {
    DTMI_CHECK(sizes[e] >= 0 && sizes[e] <= R - off[e], "%s: expert %lld has %lld rows of the %lld left", what,
               (long long)e, (long long)sizes[e], (long long)(R - off[e]));
    off[e + 1] = off[e] + sizes[e];
  }
  return DTMI_OK;
}

static const char* at(const void* p, int64_t elements, int dtype) {
  return (const char*)p + elements * (dtype == DTMI_F32 ? 4 : 8);
}
static char* at(void* p, int64_t elements, int dtype) {
  return p ? (char*)p + elements * (dtype == DTMI_F32 ? 4 : 8) : nullptr;
}

static int run(int dtype, int akc, int bkc, std::vector<GroupTask> tasks, int dmode) {
  std::vector<GroupLaunch> l;
  int rc = plan_group(dtype, akc, bkc, std::move(tasks), dmode, 0, 1.0, 0.0, 0.0, 1, 1, l);
  return rc ? rc : launch_group(dtype, l);
}

// Rows of an [R, cols] result that no expert owns: a product of no terms.
static void add_tail(int dtype, void* p, int64_t used, int64_t R, int64_t cols, std::vector<GroupTask>& t) {
  if (used < R) t.push_back({p, p, at(p, used * cols, dtype), nullptr, (int)(R - used), (int)cols, 0, 0, 1.0});
}

}  // namespace dtmi

using namespace dtmi;

DTMI_EXPORT int dtmi_expert_linear_fwd(int dtype, int64_t E, int64_t R, int64_t K, int64_t N, void* y, const void* x,
                                       const void* w, const void* b, const int64_t* sizes) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  std::vector<int64_t> off;
  int rc = expert_offsets(__func__, sizes, E, R, K, N, off);
  if (rc) return rc;
  if (R == 0 || N == 0) return DTMI_OK;
  DTMI_CHECK(y && (K == 0 || off[E] == 0 || (x && w)), "%s: NULL pointer", __func__);
  std::vector<GroupTask> t;
  for (int64_t e = 0; e < E; ++e) {
    if (off[e + 1] == off[e]) continue;
    t.push_back({at(x, off[e] * K, dtype), at(w, e * K * N, dtype), at(y, off[e] * N, dtype),
                 at(const_cast<void*>(b), e * N, dtype), (int)(off[e + 1] - off[e]), (int)N, (int)K, 0, 1.0});
  }
  add_tail(dtype, y, off[E], R, N, t);
  return run(dtype, 1, 0, std::move(t), b ? kDRow : kDNone);
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_expert_linear_bwd_dx(int dtype, int64_t E, int64_t R, int64_t K, int64_t N, void* dx,
                                          const void* g, const void* w, const int64_t* sizes) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  std::vector<int64_t> off;
  int rc = expert_offsets(__func__, sizes, E, R, K, N, off);
  if (rc) return rc;
  if (R == 0 || K == 0) return DTMI_OK;
  DTMI_CHECK(dx && (N == 0 || off[E] == 0 || (g && w)), "%s: NULL pointer", __func__);
  std::vector<GroupTask> t;
  for (int64_t e = 0; e < E; ++e) {
    if (off[e + 1] == off[e]) continue;
    t.push_back({at(g, off[e] * N, dtype), at(w, e * K * N, dtype), at(dx, off[e] * K, dtype), nullptr,
                 (int)(off[e + 1] - off[e]), (int)K, (int)N, 0, 1.0});
  }
  add_tail(dtype, dx, off[E], R, K, t);
  return run(dtype, 1, 1, std::move(t), kDNone);
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_expert_linear_bwd_dw(int dtype, int64_t E, int64_t R, int64_t K, int64_t N, void* dw, void* db,
                                          const void* x, const void* g, const int64_t* sizes) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  DTMI_DTYPE_OK(dtype);
  std::vector<int64_t> off;
  int rc = expert_offsets(__func__, sizes, E, R, K, N, off);
  if (rc) return rc;
  if (N == 0 || E == 0) return DTMI_OK;
  DTMI_CHECK(K == 0 || dw, "%s: NULL pointer", __func__);
  DTMI_CHECK(off[E] == 0 || (g && (K == 0 || x)), "%s: NULL pointer", __func__);
  if (K == 0) {  // no tiles of dw to carry db
    for (int64_t e = 0; db && e < E; ++e) {
      rc = dtmi_colsum(dtype, at(db, e * N, dtype), at(g, off[e] * N, dtype), off[e + 1] - off[e], N, 0);
      if (rc) return rc;
    }
    return DTMI_OK;
  }
  std::vector<GroupTask> t;
  for (int64_t e = 0; e < E; ++e)  // experts without rows: zeros
    t.push_back({at(x, off[e] * K, dtype), at(g, off[e] * N, dtype), at(dw, e * K * N, dtype), at(db, e * N, dtype),
                 (int)K, (int)N, (int)(off[e + 1] - off[e]), 0, 1.0});
  return run(dtype, 0, 0, std::move(t), db ? kDColsum : kDNone);
  DTMI_BODY_END
}
