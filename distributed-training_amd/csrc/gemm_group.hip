// Plans and launches of the group and statistics products (gemm_group.h).
#include "gemm_group.h"

namespace dtmi {

// SIMD cycles of a launch, as tile_cost in gemm.hip (the same constants): rounds of
// blocks x k x the MFMA time of a tile over the rate it reaches, the longest task's
// own chain at least, and a split's partials and second launch.
static double group_cost(const GroupTask* t, int count, int sym, int bm, int splits, int64_t cus, size_t es) {
  const int64_t bk = 64 / (int64_t)es;
  double work = 0, chain = 0;
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t tm = cdiv(t[i].M, bm), tn = cdiv(t[i].N, bm), n = sym ? tm * (tm + 1) / 2 : tm * tn;
    const double k = (double)(cdiv(cdiv(t[i].K, splits), bk) * bk);
    tiles += n;
    work += (double)n * k;
    if (n && k > chain) chain = k;
  }
  if (!tiles) return 0;
  const int64_t blocks = tiles * splits;
  const double rounds = (double)cdiv(blocks, cus);
  const double eff = bm == 64 ? (rounds > 1 ? 0.88 : 0.75) : rounds > 2 ? 0.97 : rounds > 1 ? 1.0 : 0.82;
  const double per_k = (es == 4 ? 32.0 : 64.0) * (bm / 32) * (bm / 32) / 4.0;  // four waves
  const double k = rounds * work / (double)tiles;
  double c = 8800.0 + (k > chain ? k : chain) * per_k / eff;
  if (splits > 1) c += 6600.0 + (double)tiles * bm * bm * (double)es * (splits + 1) / 2700.0;
  return c;
}

// The float32 sums of a 128-wide tile are one chain over its k range (64-wide tiles
// fold theirs): at most 4096 k.
static GroupPlan plan_group(const GroupTask* t, int count, int sym, int64_t cus, size_t es) {
  int kmax = 0;
  for (int i = 0; i < count; ++i) kmax = t[i].K > kmax ? t[i].K : kmax;
  GroupPlan best{64, 1};
  double least = -1;
  for (int bm = 64; bm <= 128; bm += 64)
    for (int sp = 1; sp <= 16 && (sp == 1 || kmax / sp >= 128); ++sp) {
      if (bm == 128 && es == 4 && kmax / sp > 4096 && sp < 16) continue;
      const double c = group_cost(t, count, sym, bm, sp, cus, es);
      if (least < 0 || c < least) {
        least = c;
        best = {bm, sp};
      }
    }
  return best;
}

template <typename T>
static int group_launches(int akc, int bkc, GroupTask* tasks, int count, int dmode, int sym, double alpha, double beta,
                          double gamma) {
  constexpr int V = MF<T>::VEC;
  const int64_t cus = num_cus() > 0 ? num_cus() : 256;
  for (int lo = 0; lo < count; lo += kGroupTasks) {
    GroupArgs a{};
    a.count = count - lo < kGroupTasks ? count - lo : kGroupTasks;
    a.dmode = dmode;
    a.sym = sym;
    a.alpha = alpha;
    a.beta = beta;
    a.gamma = gamma;
    bool vec = true;
    double flops = 0;
    for (int i = 0; i < a.count; ++i) {
      GroupTask& t = a.t[i];
      t = tasks[lo + i];
      const int64_t lda = akc ? t.K : t.M, ldb = bkc ? t.K : t.N;
      DTMI_CHECK(lda <= kTileMaxLd<T> && ldb <= kTileMaxLd<T> && t.N <= kTileMaxLd<T>,
                 "group of products: rows of 2^24 bytes or more are not supported");
      vec = vec && lda % V == 0 && ldb % V == 0 && aligned(t.A, 16) && aligned(t.B, 16) &&
            (!sym || (t.N % V == 0 && aligned(t.C, 16)));
      flops += (sym ? 1.0 : 2.0) * (double)t.M * t.N * t.K;
    }
    const GroupPlan p = plan_group(a.t, a.count, sym, cus, sizeof(T));
    int64_t tiles = 0;
    for (int i = 0; i < a.count; ++i) {
      const int64_t tm = cdiv(a.t[i].M, p.tile), tn = cdiv(a.t[i].N, p.tile);
      a.t[i].tile0 = (int)tiles;
      tiles += sym ? tm * (tm + 1) / 2 : tm * tn;
      DTMI_CHECK(tiles < (1LL << 30), "group of products: too large");
    }
    if (!tiles) continue;
    a.tiles = (int)tiles;
    a.splits = p.splits;
    void* ws = nullptr;
    if (p.splits > 1) {
      const size_t main_bytes = (size_t)p.splits * tiles * p.tile * p.tile * sizeof(T);
      const size_t cs_bytes = dmode == kDColsum ? (size_t)p.splits * a.count * a.t[0].N * sizeof(T) : 0;
      int rc = pool_alloc(&ws, main_bytes + cs_bytes);
      if (rc) return rc;
      a.ws = ws;
      if (cs_bytes) a.csws = (char*)ws + main_bytes;
    }
    {
      TimedLaunch tl(DTMI_FAM_GEMM, flops);
      if (p.tile == 64)
        launch_group<T, 64>(a, akc, bkc, vec);
      else
        launch_group<T, 128>(a, akc, bkc, vec);
    }
    const hipError_t e = hipGetLastError();
    if (ws) pool_free(ws);
    if (e != hipSuccess) return fail_hip(e, "group kernels", __FILE__, __LINE__);
  }
  return DTMI_OK;
}

int run_group(int dtype, int akc, int bkc, GroupTask* tasks, int count, int dmode, int sym, double alpha, double beta,
              double gamma) {
  if (dtype == DTMI_F32) return group_launches<float>(akc, bkc, tasks, count, dmode, sym, alpha, beta, gamma);
  return group_launches<double>(akc, bkc, tasks, count, dmode, sym, alpha, beta, gamma);
}

static int stats_tile(int dtype, int64_t M, int64_t N, int64_t K) {
  GroupTask t{};
  t.M = (int)M;
  t.N = (int)N;
  t.K = (int)K;
  const int64_t cus = num_cus() > 0 ? num_cus() : 256;
  const size_t es = dtype == DTMI_F32 ? 4 : 8;
  return group_cost(&t, 1, 0, 64, 1, cus, es) < group_cost(&t, 1, 0, 128, 1, cus, es) ? 64 : 128;
}

int64_t stats_parts(int dtype, int64_t M, int64_t N, int64_t K) { return 2 * cdiv(N, stats_tile(dtype, M, N, K)); }

template <typename T>
static int stats_launch(int dtype, int bkc, StatsArgs& a) {
  constexpr int V = MF<T>::VEC;
  DTMI_CHECK(a.lda <= kTileMaxLd<T> && a.ldb <= kTileMaxLd<T> && a.ldc <= kTileMaxLd<T>,
             "statistics product: rows of 2^24 bytes or more are not supported");
  const bool vec = aligned(a.A, 16) && aligned(a.B, 16) && a.lda % V == 0 && a.ldb % V == 0 && a.K % V == 0 &&
                   (bkc || a.N % V == 0);
  const int tile = stats_tile(dtype, a.M, a.N, a.K);
  DTMI_CHECK(cdiv(a.M, tile) * cdiv(a.N, tile) < (1LL << 30), "statistics product: too large");
  a.tiles_m = (int)cdiv(a.M, tile);
  a.tiles_n = (int)cdiv(a.N, tile);
  {
    TimedLaunch tl(DTMI_FAM_GEMM, 2.0 * (double)a.M * a.N * a.K);
    if (tile == 64)
      launch_stats<T, 64>(a, bkc, vec);
    else
      launch_stats<T, 128>(a, bkc, vec);
  }
  LAUNCH_CHECK("gemm_stats_kernel");
  return DTMI_OK;
}

int run_stats(int dtype, int bkc, StatsArgs a) {
  return dtype == DTMI_F32 ? stats_launch<float>(dtype, bkc, a) : stats_launch<double>(dtype, bkc, a);
}

}  // namespace dtmi
