// Shared by the sequence operators over [B, T, C] activations (conv.hip,
// scan.hip): row vectors of a thread's channels and the activations.
#pragma once

#include <cmath>

#include "common.h"

namespace dtmi {

// Element strides of the batch and time axes of a [B, T, C] array (C contiguous).
struct BT {
  int64_t b, t;
};

template <typename T, int VW>
__device__ __forceinline__ void vload(T (&x)[VW], const T* __restrict__ p) {
  typedef T vt __attribute__((ext_vector_type(VW == 1 ? 2 : VW)));
  if constexpr (VW == 1) {
    x[0] = p[0];
  } else {
    const vt v = *reinterpret_cast<const vt*>(p);
#pragma unroll
    for (int e = 0; e < VW; ++e) x[e] = v[e];
  }
}
template <typename T, int VW>
__device__ __forceinline__ void vstore(T* __restrict__ p, const T (&x)[VW]) {
  typedef T vt __attribute__((ext_vector_type(VW == 1 ? 2 : VW)));
  if constexpr (VW == 1) {
    p[0] = x[0];
  } else {
    vt v;
#pragma unroll
    for (int e = 0; e < VW; ++e) v[e] = x[e];
    *reinterpret_cast<vt*>(p) = v;
  }
}

// 2^x: one v_exp_f32 in float32, the accurate library routine in float64.
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double exp2_of(double x) { return exp2(x); }

// 1 / (1 + exp(-x)). float32: the base-2 exponential and reciprocal of the
// hardware, about 1 ulp each; the argument's rounding costs |x| 2^-24 of the
// small side, where the value itself is below exp(-|x|).
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}
// 1 / x for 1 <= x < 2^1020: the hardware's approximation and two Newton steps.
__device__ __forceinline__ double rcp_of(double x) {
  double r = __builtin_amdgcn_rcp(x);
  r = fma(fma(-x, r, 1.0), r, r);
  return fma(fma(-x, r, 1.0), r, r);
}
// (below -700 the value stays at exp(-700), so that 1 + exp(-x) is finite)
__device__ __forceinline__ double sigmoid(double x) { return rcp_of(1.0 + exp(x < -700.0 ? 700.0 : -x)); }

// log(1 + exp(x)) = max(x, 0) + log1p(exp(-|x|)). Step sizes of 1e-3 live in
// the second term, so it needs its relative accuracy: log1p(e) = 2 atanh(s) with
// s = e / (2 + e) <= 1/3, whose series ends below 2^-25 after s^14 / 15.
__device__ __forceinline__ float softplus(float x) {
  const float e = __builtin_amdgcn_exp2f(fabsf(x) * -1.44269504f);
  const float s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
  float r = 1.f / 15.f;
  r = fmaf(r, q, 1.f / 13.f);
  r = fmaf(r, q, 1.f / 11.f);
  r = fmaf(r, q, 1.f / 9.f);
  r = fmaf(r, q, 1.f / 7.f);
  r = fmaf(r, q, 1.f / 5.f);
  r = fmaf(r, q, 1.f / 3.f);
  r = fmaf(r, q, 1.f);
  // the maximum as a comparison that is false for NaN would lose it: x + 0 keeps it
  return (x < 0.f ? 0.f : x) + 2.f * s * r;
}
// the same in float64: the series ends below 2^-55 after s^32 / 33 (3 x 257 x 384 x 8
// forward and backward, where a wave stages four rows a tile: kernels 89 us with the
// library's logarithm and division, 77 so)
__device__ __forceinline__ double softplus(double x) {
  const double e = exp(-fabs(x)), s = e * rcp_of(2.0 + e), q = s * s;
  double r = 1.0 / 33.0;
#pragma unroll
  for (int k = 31; k > 0; k -= 2) r = fma(r, q, 1.0 / k);
  return (x < 0.0 ? 0.0 : x) + 2.0 * s * r;
}

// Positions of a sequence that hold data: lengths[b] within [0, T], or all.
__device__ __forceinline__ int64_t seq_len(const int64_t* __restrict__ lengths, int64_t b, int64_t T) {
  if (!lengths) return T;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n > T ? T : n;
}

}  // namespace dtmi
