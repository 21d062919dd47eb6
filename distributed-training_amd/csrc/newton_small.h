// Newton-Schulz steps of small matrices, one block each, and of thin ones, a block for
// each 64 columns (newton_small.hip).
#pragma once

#include "gemm_common.h"

namespace dtmi {

constexpr int kSmallTasks = 64;  // 48 bytes each: the arguments stay below 4 KB

struct SmallTask {
  const void* g;
  void* m;    // momentum (NULL: u = g)
  void* out;  // gamma out + rate X
  double rate;
  int rows, cols;
};

struct SmallArgs {
  int steps, nesterov;
  double a, b, c, eps, mu, gscale, gamma;
  const double* gscale_dev;
  SmallTask t[kSmallTasks];
};

enum ThinStage { kThinFirst, kThinStep, kThinLast };

struct ThinTask {
  const void* g;
  void* m;    // momentum, moved on (NULL: u = g)
  void* out;  // gamma out + rate X
  void* ws;   // thin_bytes
  double rate;
  int rows, cols;
  int first;  // the matrix's first block
};

struct ThinArgs {
  int count, stage, nesterov;
  int at, part_count;   // the first matrix's number; parts of each matrix's sum of squares
  const double* parts;  // [matrices][part_count]
  double a, b, c, eps, mu, gscale, gamma;
  const double* gscale_dev;
  ThinTask t[kSmallTasks];
};

// The most LDS of a matrix, in bytes, and the SIMD cycles its block takes for `steps` steps.
int64_t small_lds(int dtype, int64_t rows, int64_t cols);
double small_cycles(int dtype, int64_t rows, int64_t cols, int steps);
// The most LDS a block may have.
int64_t small_lds_limit();
int launch_small(int dtype, const SmallArgs& a, int count);
// Of a thin matrix: LDS, workspace, blocks, and the cycles of one step of a launch of `blocks`.
int64_t thin_lds(int dtype, int64_t rows, int64_t cols);
int64_t thin_bytes(int dtype, int64_t rows, int64_t cols);
int64_t thin_blocks(int64_t rows, int64_t cols);
double thin_cycles(int dtype, int64_t rows, int64_t cols, int64_t blocks, int64_t cus);
// blocks: of the stage's launch; 0: the joins.
int launch_thin(int dtype, const ThinArgs& a, int blocks);

}  // namespace dtmi
