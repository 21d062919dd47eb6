// Plans and launches of the group and statistics products (gemm_group.h).
#include "gemm_group.h"

#include <algorithm>

#include "gemm_direct.h"
#include "gemm_rows.h"

namespace dtmi {

// Block tile (32: the small-product kernels, of nw waves), and how many tiles of a launch
// are split along k (kAll: all).
constexpr int kAll = 1 << 30;
struct GroupPlan {
  int tile, cut, splits, nw;
};

// Few rows: gemm_rows.h, up to 32 (the tile is then 16 or 32 rows).
constexpr int kFewRows = 32;

// Bytes of a wave's tile of few rows.
template <typename T>
static int64_t rows_bytes(int mr, int bkc) {
  return 4 * mr * (bkc ? RowsTile<T, true>::NT : RowsTile<T, false>::NT) * 64 * (int64_t)sizeof(T);
}

// Waves of a block of few rows: 16 per CU, each with at least a batch of k, and their
// partial tiles within 64 KB.
template <typename T>
static int rows_waves(int64_t blocks, int64_t K, int64_t cus, int mr, int bkc) {
  const int64_t bytes = rows_bytes<T>(mr, bkc);
  int64_t w = 1;
  while (w < kRowsMaxWaves && blocks * w < 16 * cus && 2 * w * bytes <= 64 * 1024) w *= 2;
  const int64_t batches = cdiv(K > 0 ? K : 1, RowsTile<T, true>::BATCH);
  return (int)(w < batches ? w : batches);
}

// Blocks along k for few rows: a wave waits about 1.8 us for each batch of its share, and
// joining the pieces is a launch of 6 us. Pieces of three batches from seven on, up to four
// blocks a CU: one row of 3993 x 136 31 -> 12 us, two of 23011 x 1247 71 (the GEMM) -> 35.
template <typename T>
static int rows_splits(int64_t blocks, int64_t K, int64_t cus, int nw) {
  const int64_t batches = cdiv(K, (int64_t)nw * RowsTile<T, true>::BATCH);
  const int64_t want = cdiv(batches, 3), fit = 4 * cus / blocks;
  const int64_t s = want < fit ? want : fit;
  return batches > 6 && s > 1 ? (int)s : 1;
}

// Waves of a small-product block: 8 per CU, each with at least a batch of k.
template <typename T>
static int direct_waves(int64_t tiles, int64_t K, int64_t cus) {
  int64_t w = 4;
  while (w < 8 && tiles * w < 8 * cus) w *= 2;
  const int64_t batches = cdiv(K > 0 ? K : 1, kDirectBatch<T>);
  return (int)(w < batches ? w : batches);
}

// SIMD cycles of a small-product launch: as direct_cost in gemm.hip.
template <typename T>
static double direct_cycles(int64_t tiles, double kavg, int64_t kmax, int nw, int64_t cus) {
  const double kps = (double)(cdiv(cdiv(kmax, nw), kDirectBatch<T>) * kDirectBatch<T>);
  const double rate = (double)cdiv(tiles, cus) * kavg * (sizeof(T) == 4 ? 8.0 / 0.45 : 16.0 / 0.55);
  const double chain = 3500.0 + 1.35 * (sizeof(T) == 4 ? 32.0 : 64.0) * kps;
  return 7700.0 + (rate > chain ? rate : chain);
}

// SIMD cycles of `units` blocks on BM-wide tiles, the busiest CU's k being `k`: as
// tile_cost in gemm.hip (64-wide float32 tiles over several tasks reach less, 0.80 to
// 0.89 of their MFMA rate), with what a block costs before its first MFMA and after its
// last, of which the others on its CU hide some: 64 experts' dw, 384 x 501 from 62 rows
// each, took 42 us on 48 64-wide tiles an expert. A 128-wide float32 tile alone on its CU waits for
// its loads, of single elements the more (vec false): four times 713 x 1075 with 619 terms,
// 216 tiles: 55 us (816 64-wide ones: 48), 704 x 1088 with 640: 48 us.
static double tile_cycles(int bm, double k, double units, int64_t cus, size_t es, bool vec) {
  const double alone = es == 8 ? 0.82 : vec ? 0.78 : 0.66;
  const double eff = bm == 64           ? (units > cus ? (es == 4 ? 0.82 : 0.88) : 0.75)
                     : units > 2.0 * cus ? 0.97
                     : units > cus       ? 1.0
                                         : alone;
  return 8800.0 + 1500.0 * units / (double)cus + k * (es == 4 ? 32.0 : 64.0) * (bm / 32) * (bm / 32) / 4.0 / eff;
}
// and what a split adds: its partials' traffic and a launch
static double split_cycles(int bm, int64_t cut, int splits, size_t es) {
  return splits > 1 ? 6600.0 + (double)cut * bm * bm * (double)es * (splits + 1) / 2700.0 : 0.0;
}

// How to run the tasks (longest k first). Blocks are dealt out as slots come free, so a
// ragged last round, or a task that outlasts the others, leaves CUs idle:
// - equal k: all tiles split (few tiles), or only as many as make the rest a whole
//   number of rounds;
// - unequal k: the tiles of the longest tasks split.
template <typename T>
static GroupPlan choose_plan(const GroupTask* t, int count, int sym, int pad, int64_t cus, bool vec) {
  constexpr size_t es = sizeof(T);
  constexpr int64_t bk = 64 / (int64_t)es;
  int64_t k[kGroupTasks];
  for (int i = 0; i < count; ++i) k[i] = cdiv(cdiv(t[i].K, pad) * pad, bk) * bk;
  GroupPlan best{64, 0, 1, 0};
  double least = -1;
  auto take = [&](double c, GroupPlan p) {
    if (least < 0 || c < least) {
      least = c;
      best = p;
    }
  };
  auto tiles_of = [&](int i, int bm) {
    if (k[i] == 0) return (int64_t)0;  // these only write
    const int64_t tm = cdiv(t[i].M, bm), tn = cdiv(t[i].N, bm);
    return sym ? tm * (tm + 1) / 2 : tm * tn;
  };
  for (int bm = 64; bm <= 128; bm += 64) {
    int64_t n[kGroupTasks], total = 0;
    double work = 0;
    int last = 0;
    for (int i = 0; i < count; ++i) {
      n[i] = tiles_of(i, bm);
      total += n[i];
      work += (double)n[i] * (double)k[i];
      if (n[i]) last = i;
    }
    if (!total) return best;
    while (last > 0 && (k[last] == 0 || n[last] == 0)) --last;  // the shortest with anything to add up
    const bool equal = k[0] == k[last];
    // one chain of float32 sums: at most 4096 k on 128-wide tiles (64-wide ones fold theirs)
    const int64_t chain = bm == 128 && es == 4 ? 4096 : 1LL << 40;
    const double even = work / (double)cus;
    if (k[0] <= chain) {
      const double busy = equal ? (double)cdiv(total, cus) * (double)k[0]
                                : std::max((double)k[0], even + 0.5 * (double)k[last]);
      take(tile_cycles(bm, busy, (double)total, cus, es, vec), {bm, 0, 1, 0});
    }
    const int64_t rest = equal && total > cus ? total % cus : 0;
    for (int sp = 2; sp <= 16 && k[0] / sp >= 128; ++sp) {
      const double ks = (double)(cdiv(cdiv(k[0], sp), bk) * bk);
      if (ks <= (double)chain || sp == 16) {
        const double busy =
            equal ? (double)cdiv(total * sp, cus) * ks : std::max(ks, even + 0.5 * (double)k[last] / sp);
        take(tile_cycles(bm, busy, (double)(total * sp), cus, es, vec) + split_cycles(bm, total, sp, es),
             {bm, kAll, sp, 0});
      }
      if (rest && k[0] <= chain) {
        // a quarter tile more: the last whole tiles run beside fewer and fewer pieces
        const double busy = ((double)(total / cus) + 0.25) * (double)k[0] + (double)cdiv(rest * sp, cus) * ks;
        take(tile_cycles(bm, busy, (double)(total + rest * (sp - 1)), cus, es, vec) + split_cycles(bm, rest, sp, es),
             {bm, (int)rest, sp, 0});
      }
      if (!equal && (sp <= 4 || sp % 4 == 0)) {
        int64_t cut = 0;
        for (int i = 0; i < last && i < 16; ++i) {
          cut += n[i];
          if (k[i] == k[i + 1] || !cut || k[i + 1] > chain || ks > (double)chain) continue;
          const double busy = std::max(std::max(ks, (double)k[i + 1]), even + 0.5 * (double)k[last]);
          take(tile_cycles(bm, busy, (double)(total + cut * (sp - 1)), cus, es, vec) + split_cycles(bm, cut, sp, es),
               {bm, (int)cut, sp, 0});
        }
      }
    }
  }
  int64_t tiles = 0;
  double work = 0;
  for (int i = 0; i < count; ++i) {
    tiles += tiles_of(i, 32);
    work += (double)tiles_of(i, 32) * (double)k[i];
  }
  const int nw = direct_waves<T>(tiles, k[0], cus);
  take(direct_cycles<T>(tiles, work / (double)tiles, k[0], nw, cus), {32, 0, 1, nw});
  return best;
}

template <typename T>
static int plan_tasks(int akc, int bkc, std::vector<GroupTask>& tasks, int dmode, int sym, double alpha, double beta,
                      double gamma, int pad, int padc, std::vector<GroupLaunch>& out) {
  constexpr int V = MF<T>::VEC;
  const int64_t cus = num_cus() > 0 ? num_cus() : 256;
  const int count = (int)tasks.size();
  std::stable_sort(tasks.begin(), tasks.end(), [](const GroupTask& x, const GroupTask& y) { return x.K > y.K; });
  for (int lo = 0; lo < count; lo += kGroupTasks) {
    GroupLaunch l{};
    GroupArgs& a = l.a;
    l.akc = akc;
    l.bkc = bkc;
    a.count = count - lo < kGroupTasks ? count - lo : kGroupTasks;
    a.dmode = dmode;
    a.sym = sym;
    a.pad = pad;
    a.padc = padc;
    a.alpha = alpha;
    a.beta = beta;
    a.gamma = gamma;
    bool vec = true;
    int rows = 0;
    for (int i = 0; i < a.count; ++i) {
      GroupTask& t = a.t[i];
      t = tasks[lo + i];
      const int64_t lda = cdiv(akc ? t.K : t.M, pad) * pad, ldb = cdiv(bkc ? t.K : t.N, pad) * pad;
      DTMI_CHECK(lda <= kTileMaxLd<T> && ldb <= kTileMaxLd<T> && t.N <= kTileMaxLd<T>,
                 "group of products: rows of 2^24 bytes or more are not supported");
      vec = vec && lda % V == 0 && ldb % V == 0 && aligned(t.A, 16) && aligned(t.B, 16) &&
            (!sym || (cdiv(t.N, padc) * padc % V == 0 && aligned(t.C, 16)));
      if (t.K > 0 && t.M > rows) rows = t.M;  // (products of no terms only write)
      l.flops += (sym ? 1.0 : 2.0) * (double)t.M * t.N * t.K;
    }
    l.vec = vec;
    const bool few = rows <= kFewRows && akc && !sym && pad == 1 && dmode != kDColsum;
    const GroupPlan p = few ? GroupPlan{16, 0, 1, 0} : choose_plan<T>(a.t, a.count, sym, pad, cus, vec);
    l.tile = p.tile;
    l.nw = p.nw;
    l.mr = rows <= 16 ? 1 : 2;
    const int tm_rows = few ? 16 * l.mr : p.tile;
    const int tn_cols = few ? (bkc ? RowsTile<T, true>::COLS : RowsTile<T, false>::COLS) : p.tile;
    a.equal = 1;
    int64_t tiles = 0, work = 0;
    for (int i = 0; i < a.count; ++i) {
      const int64_t tm = cdiv(a.t[i].M, tm_rows), tn = cdiv(a.t[i].N, tn_cols);
      a.equal = a.equal && (a.t[i].K == a.t[0].K || a.t[i].K == 0);
      a.first[i] = (int)tiles;
      tiles += sym ? tm * (tm + 1) / 2 : tm * tn;
      if (a.t[i].K > 0) work = tiles;
      DTMI_CHECK(tiles < (1LL << 26), "group of products: too large");
    }
    if (!tiles) continue;
    a.tiles = (int)tiles;
    a.work = (int)work;
    if (few) l.nw = rows_waves<T>(tiles, a.t[0].K, cus, l.mr, bkc);
    const int pieces = few ? rows_splits<T>(tiles, a.t[0].K, cus, l.nw) : p.splits;
    a.cut = p.cut < a.work ? p.cut : a.work;
    a.splits = pieces;
    for (int i = 0; i < a.count && a.cut; ++i) {  // whole tiles that are longer than the pieces
      const int end = i + 1 < a.count ? a.first[i + 1] : a.tiles;
      if (end > a.cut && a.t[i].K > 0 && a.t[i].K >= cdiv(a.t[0].K, p.splits)) a.before = end - a.cut;
    }
    if (!a.equal && p.tile == 128) {  // the blocks that have something to do, longest first
      const int64_t units = a.work + (int64_t)a.cut * (p.splits - 1);
      if (units > cus && units <= 2 * cus) {
        a.turn = (int)cus;
        a.turned = (int)units;
      }
    }
    if (few && pieces > 1) l.ws_bytes = (size_t)pieces * tiles * rows_bytes<T>(l.mr, bkc);
    if (a.cut) {
      const size_t slots = (size_t)p.splits * a.cut;
      l.cs_at = slots * p.tile * p.tile * sizeof(T);
      l.ws_bytes = l.cs_at + (dmode == kDColsum ? slots * p.tile * sizeof(T) : 0);
    }
    out.push_back(l);
  }
  return DTMI_OK;
}

int plan_group(int dtype, int akc, int bkc, std::vector<GroupTask> tasks, int dmode, int sym, double alpha, double beta,
               double gamma, int pad, int padc, std::vector<GroupLaunch>& out) {
  out.clear();
  if (dtype == DTMI_F32) return plan_tasks<float>(akc, bkc, tasks, dmode, sym, alpha, beta, gamma, pad, padc, out);
  return plan_tasks<double>(akc, bkc, tasks, dmode, sym, alpha, beta, gamma, pad, padc, out);
}

template <typename T>
static int launch_one(const GroupLaunch& l) {
  void* ws = nullptr;
  GroupArgs a = l.a;
  if (l.ws_bytes) {
    int rc = pool_alloc(&ws, l.ws_bytes);
    if (rc) return rc;
    a.ws = ws;
    a.csws = (char*)ws + l.cs_at;
  }
  {
    TimedLaunch tl(DTMI_FAM_GEMM, l.flops);
    if (l.tile == 16)
      launch_group_rows<T>(a, l.bkc, l.mr, l.nw);
    else if (l.tile == 32)
      launch_group_direct<T>(a, l.akc, l.bkc, l.nw);
    else if (l.tile == 64)
      launch_group<T, 64>(a, l.akc, l.bkc, l.vec);
    else
      launch_group<T, 128>(a, l.akc, l.bkc, l.vec);
  }
  const hipError_t e = hipGetLastError();
  if (ws) pool_free(ws);
  if (e != hipSuccess) return fail_hip(e, "group kernels", __FILE__, __LINE__);
  return DTMI_OK;
}

int launch_group(int dtype, const std::vector<GroupLaunch>& launches) {
  for (const GroupLaunch& l : launches) {
    int rc = dtype == DTMI_F32 ? launch_one<float>(l) : launch_one<double>(l);
    if (rc) return rc;
  }
  return DTMI_OK;
}

// What the statistics of a tile add to its product (exponentials, and the joins along its
// rows): a block alone on its CU waits for all of it, the others hide two thirds. float32
// 388 x 17704 with 66 terms: 42.8 us on 32-wide tiles, 24.2 on 64, 24.9 on 128; float64
// 3224 x 161 with 339 terms: 19.8, 22.6 and 57.9.
static double epilogue_cycles(int bm, int64_t units, int64_t cus, size_t es) {
  const double one = es == 4 ? (bm == 128 ? 15000.0 : bm == 64 ? 5000.0 : 6000.0)
                             : (bm == 128 ? 23000.0 : bm == 64 ? 15000.0 : 7000.0);
  return one * (1.0 + 0.35 * (double)(cdiv(units, cus) - 1));
}

// Tile and waves of a statistics product (tile 16: few rows).
template <typename T>
static GroupPlan plan_stats(int bkc, int64_t M, int64_t N, int64_t K) {
  const int64_t cus = num_cus() > 0 ? num_cus() : 256;
  if (M <= kFewRows) {
    const int64_t blocks = cdiv(N, bkc ? RowsTile<T, true>::COLS : RowsTile<T, false>::COLS);
    return {16, 0, 1, rows_waves<T>(blocks, K, cus, M <= 16 ? 1 : 2, bkc)};
  }
  constexpr int64_t bk = 64 / (int64_t)sizeof(T);
  const double k = (double)(cdiv(K, bk) * bk);
  const int64_t t32 = cdiv(M, 32) * cdiv(N, 32);
  GroupPlan best{32, 0, 1, direct_waves<T>(t32, K, cus)};
  double least = direct_cycles<T>(t32, (double)K, K, best.nw, cus) + epilogue_cycles(32, t32, cus, sizeof(T));
  for (int bm = 64; bm <= 128; bm += 64) {
    const int64_t n = cdiv(M, bm) * cdiv(N, bm);
    const double c = tile_cycles(bm, (double)cdiv(n, cus) * k, (double)n, cus, sizeof(T), true) +
                     epilogue_cycles(bm, n, cus, sizeof(T));
    if (c < least) {
      least = c;
      best = {bm, 0, 1, 0};
    }
  }
  return best;
}

template <typename T>
static int64_t parts_of(const GroupPlan& p, int bkc, int64_t N) {
  if (p.tile == 16) return cdiv(N, bkc ? RowsTile<T, true>::COLS : RowsTile<T, false>::COLS);
  // a wave's columns: MFMA tiles of 32, or half a block tile
  return p.tile == 32 ? cdiv(N, 32) * (32 / MF<T>::MT) : 2 * cdiv(N, p.tile);
}

int64_t stats_parts(int dtype, int bkc, int64_t M, int64_t N, int64_t K) {
  return dtype == DTMI_F32 ? parts_of<float>(plan_stats<float>(bkc, M, N, K), bkc, N)
                           : parts_of<double>(plan_stats<double>(bkc, M, N, K), bkc, N);
}

template <typename T>
static int stats_launch(int bkc, StatsArgs& a) {
  constexpr int V = MF<T>::VEC;
  DTMI_CHECK(a.lda <= kTileMaxLd<T> && a.ldb <= kTileMaxLd<T> && a.ldc <= kTileMaxLd<T>,
             "statistics product: rows of 2^24 bytes or more are not supported");
  const GroupPlan p = plan_stats<T>(bkc, a.M, a.N, a.K);
  const bool vec = aligned(a.A, 16) && aligned(a.B, 16) && a.lda % V == 0 && a.ldb % V == 0 && a.K % V == 0 &&
                   (bkc || a.N % V == 0);
  DTMI_CHECK(cdiv(a.M, p.tile) * cdiv(a.N, p.tile) < (1LL << 30), "statistics product: too large");
  const int mr = a.M <= 16 ? 1 : 2;
  a.tiles_m = p.tile == 16 ? 1 : (int)cdiv(a.M, p.tile);
  a.tiles_n = (int)(p.tile == 16 ? parts_of<T>(p, bkc, a.N) : cdiv(a.N, p.tile));
  {
    TimedLaunch tl(DTMI_FAM_GEMM, 2.0 * (double)a.M * a.N * a.K);
    if (p.tile == 16)
      launch_stats_rows<T>(a, bkc, mr, p.nw);
    else if (p.tile == 32)
      launch_stats_direct<T>(a, bkc, p.nw);
    else if (p.tile == 64)
      launch_stats<T, 64>(a, bkc, vec);
    else
      launch_stats<T, 128>(a, bkc, vec);
  }
  LAUNCH_CHECK("statistics kernels");
  return DTMI_OK;
}

int run_stats(int dtype, int bkc, StatsArgs a) {
  return dtype == DTMI_F32 ? stats_launch<float>(bkc, a) : stats_launch<double>(bkc, a);
}

}  // namespace dtmi
