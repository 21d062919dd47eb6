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
__device__ __forceinline__ double sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }

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
__device__ __forceinline__ double softplus(double x) { return (x < 0.0 ? 0.0 : x) + log1p(exp(-fabs(x))); }

// Positions of a sequence that hold data: lengths[b] within [0, T], or all.
__device__ __forceinline__ int64_t seq_len(const int64_t* __restrict__ lengths, int64_t b, int64_t T) {
  if (!lengths) return T;
  const int64_t n = lengths[b];
  return n < 0 ? 0 : n > T ? T : n;
}

}  // namespace dtmi
