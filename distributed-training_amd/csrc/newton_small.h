// Newton-Schulz steps of small matrices, one block each (newton_small.hip).
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

// The most LDS of a matrix, in bytes, and the SIMD cycles its block takes for `steps` steps.
int64_t small_lds(int dtype, int64_t rows, int64_t cols);
double small_cycles(int dtype, int64_t rows, int64_t cols, int steps);
// The most LDS a block may have.
int64_t small_lds_limit();
int launch_small(int dtype, const SmallArgs& a, int count);

}  // namespace dtmi
