// Products of a group of matrices in one launch, and a product that keeps only row
// statistics, on the block tiles of gemm_tiles.h. Declarations and launches;
// gemm_group_tiles.h holds the kernels.
//
// A group is up to 64 tasks C = s (alpha A B + beta D) + gamma C of sizes of their
// own, passed by value with the launch: experts with the rows they were given, or
// the matrices that one optimizer step updates. Block b of the launch takes tile b
// of the tasks laid end to end; there is no table to upload and none to outlive a
// captured graph.
#pragma once

#include "gemm_common.h"

namespace dtmi {

constexpr int kGroupTasks = 64;  // 56 bytes each: the arguments stay below 4 KB

// Row-major matrices without gaps: A is [M, K] or, where m is contiguous, [K, M]; B is
// [K, N] or, where k is contiguous, [N, K]; C is [M, N].
struct GroupTask {
  const void* A;
  const void* B;
  void* C;
  void* D;
  int M, N, K;
  int tile0;  // the launch's first tile of this task
  double s;
};

// What D is: nothing, [M, N] (times beta), a row [N] added to every row, or where the
// column sums of B over k go ([N], the bias gradient of dW = X^T dY).
enum GroupD { kDNone = 0, kDMatrix = 1, kDRow = 2, kDColsum = 3 };

struct GroupArgs {
  int count, tiles, splits, dmode;
  int sym;    // A B is symmetric (M = N): tiles on and below the diagonal, the others mirrored
  void* ws;   // split-K partials, [splits][tiles][BM * BN] (NULL when not split)
  void* csws; // and the column sums' [splits][count][N]
  double alpha, beta, gamma;
  GroupTask t[kGroupTasks];
};

// Row statistics of Z = A B + bias over pieces of its columns, without Z (or with it,
// where C is not NULL): part p of row m covers half a block tile's columns, pmax[p M +
// m] is their maximum and psum[p M + m] the sum of exp(z - pmax) over them; zt[m] = Z[m,
// targets[m]].
struct StatsArgs {
  const void* A;
  const void* B;
  const void* bias;
  void* C;
  void* pmax;
  void* psum;
  void* zt;
  const int64_t* targets;
  int64_t M, N, K, lda, ldb, ldc;
  int tiles_m, tiles_n;
};

// Block tile of a launch over these tasks (64 or 128) and its k splits, by the
// estimate that gemm.hip makes of a single product.
struct GroupPlan {
  int tile, splits;
};

// gemm_group_f32.hip, gemm_group_f64.hip: one tile and type each
template <typename T, int BM>
void launch_group(const GroupArgs& a, int akc, int bkc, bool vec);
template <typename T, int BM>
void launch_stats(const StatsArgs& a, int bkc, bool vec);

// The tasks (their tile0 unset) as one launch per 64 of them, with the sum pass of a
// split. akc, bkc: which operands are k-contiguous (1, 0), (1, 1) or (0, 0).
int run_group(int dtype, int akc, int bkc, GroupTask* tasks, int count, int dmode, int sym, double alpha, double beta,
              double gamma);
// The parts a row's statistics come in.
int64_t stats_parts(int dtype, int64_t M, int64_t N, int64_t K);
int run_stats(int dtype, int bkc, StatsArgs a);

// Leading dimensions the tile kernels address (their byte offsets are 32 bits wide).
template <typename T>
constexpr int64_t kTileMaxLd = (1 << 24) / (int64_t)sizeof(T) - 1;

}  // namespace dtmi
