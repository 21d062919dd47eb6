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

#include <vector>

#include "gemm_common.h"

namespace dtmi {

constexpr int kGroupTasks = 64;  // 56 bytes each: the arguments stay below 4 KB

// Row-major matrices: A is [M, K] or, where m is contiguous, [K, M]; B is [K, N] or,
// where k is contiguous, [N, K]; C is [M, N]. See GroupArgs for their rows' lengths.
struct GroupTask {
  const void* A;
  const void* B;
  void* C;
  void* D;
  int M, N, K;
  int turned;  // C is written transposed, [N, M]
  double s;
};

// What D is: nothing, [M, N] (times beta), a row [N] added to every row, or where the
// column sums of B over k go ([N], the bias gradient of dW = X^T dY).
enum GroupD { kDNone = 0, kDMatrix = 1, kDRow = 2, kDColsum = 3 };

// The order of the blocks. At a launch's start the dispatcher goes round the CUs, one
// block each; later it fills whatever slots are free, two on one CU if need be, without
// regard to how long they will take. So the longest go first, and the pieces of split tiles
// among them by their length. Blocks are dealt to the 8 XCDs in turn; where all tasks have
// one k (`equal`), each XCD gets neighbouring tiles, an eighth of the launch, and shares
// their operands in its L2; where they differ that would give one XCD all of the longest
// task (8 experts' dw 305 us), and tiles go round as they are numbered.
struct GroupArgs {
  int count, tiles;
  // The tiles with something to add up, which come first; dealt to the XCDs in ranges where
  // all of those are equally long. The others, zeros alone, follow in their own order: in
  // the ranges they left one XCD idle in eight (2854 rows of four experts and 713 of none,
  // 619 x 1075: 58 us instead of 48).
  int work, equal;
  // the first `cut` tiles are split in `splits` along k, their partials added by a second
  // kernel; `before` blocks of whole tiles run before them
  int cut, splits, before;
  // blocks turn .. turned - 1 in reverse (none: both 0): with one round and some of the
  // next, the shortest then come to lie beside the longest
  int turn, turned;
  int dmode;
  int sym;        // A B is symmetric (M = N): tiles on and below the diagonal, the others mirrored
  // A, B and D have both dimensions rounded up to `pad`, with zeros there; C to padc, and
  // the zeros are written where padc = pad. 1: matrices without gaps.
  int pad, padc;
  void* ws;       // [splits][cut][BM * BM] partials
  void* csws;     // and the column sums' [splits][cut][BM]
  double alpha, beta, gamma;
  int first[kGroupTasks];  // each task's first tile
  GroupTask t[kGroupTasks];
};

// Row statistics of Z = A B + bias over pieces of its columns, without Z (or with it,
// where C is not NULL): part p of row m covers some columns (half a block tile's), pmax[p
// M + m] is their maximum and psum[p M + m] the sum of exp(z - pmax) over them; zt[m] =
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

// gemm_group_f32.hip, ...: one tile and type each; BM = 32: operands straight to
// registers, k over the `nw` waves of a block (gemm_direct.hip)
template <typename T, int BM>
void launch_group(const GroupArgs& a, int akc, int bkc, bool vec);
template <typename T, int BM>
void launch_stats(const StatsArgs& a, int bkc, bool vec);
template <typename T>
void launch_group_direct(const GroupArgs& a, int akc, int bkc, int nw);
template <typename T>
void launch_stats_direct(const StatsArgs& a, int bkc, int nw);
// tiles of 16 mr rows (gemm_rows.h), A k-contiguous
template <typename T>
void launch_group_rows(const GroupArgs& a, int bkc, int mr, int nw);
template <typename T>
void launch_stats_rows(const StatsArgs& a, int bkc, int mr, int nw);

// One planned launch. tile: 128, 64, 32 (of nw waves) or 16 (few rows: mr tiles of 16).
struct GroupLaunch {
  GroupArgs a;
  int akc, bkc, vec, tile, nw, mr;
  size_t ws_bytes, cs_at;
  double flops;
};
// Plans the tasks' launches, longest k first, 64 to a launch. akc, bkc: which operands
// are k-contiguous: (1, 0), (1, 1) or (0, 0).
int plan_group(int dtype, int akc, int bkc, std::vector<GroupTask> tasks, int dmode, int sym, double alpha, double beta,
               double gamma, int pad, int padc, std::vector<GroupLaunch>& out);
int launch_group(int dtype, const std::vector<GroupLaunch>& launches);
// The parts a row's statistics come in.
int64_t stats_parts(int dtype, int bkc, int64_t M, int64_t N, int64_t K);
int run_stats(int dtype, int bkc, StatsArgs a);

// Leading dimensions the tile kernels address (their byte offsets are 32 bits wide).
template <typename T>
constexpr int64_t kTileMaxLd = (1 << 24) / (int64_t)sizeof(T) - 4;

}  // namespace dtmi
