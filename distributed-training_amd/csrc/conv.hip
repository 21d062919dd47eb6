// Short causal convolution over time, each channel by itself:
//   pre[t, c] = b[c] + sum_k w[k, c] x[t - K + 1 + k, c],   y = silu(pre) or pre
// over [B, T, C] activations (C contiguous), K taps of 1 to 8, positions before
// the first taken from a state [B, K - 1, C] (zeros without one).
//
// Bound: memory. A forward reads x and writes y, a backward reads x and g and
// writes dx (pre is formed again: K products against 4 or 8 bytes). A thread
// owns VW neighbouring channels (16 bytes) over SEG positions and keeps the K
// rows of its window in registers, so a row is loaded once per segment (and
// K - 1 rows twice, from L2).
#include "seqmath.h"

namespace dtmi {

struct ConvArgs {
  void *y, *state_out, *dx, *dstate, *parts;
  const void *x, *w, *b, *state, *g;
  const int64_t* lengths;
  BT sx, sy, sg, sdx;
  int64_t B, T, C, cv, nseg;  // cv: vectors of channels per row
  int seg, silu;
};

constexpr int kConvUnroll = 4;  // rows loaded together

// Row t of the input as the window sees it: the state before the first
// position, zeros at and after the sequence's end.
template <typename T, int K, int VW>
__device__ __forceinline__ void conv_row(T (&r)[VW], const ConvArgs& a, const T* __restrict__ xb, int64_t b, int64_t t,
                                         int64_t len, int64_t c) {
  if (t >= 0 && t < len) {
    vload<T, VW>(r, xb + t * a.sx.t);
  } else if (t < 0 && a.state && t >= 1 - K) {
    vload<T, VW>(r, (const T*)a.state + (b * (K - 1) + (K - 1 + t)) * a.C + c);
  } else {
#pragma unroll
    for (int e = 0; e < VW; ++e) r[e] = T(0);
  }
}

// 8 x 1024 x 1536, 4 taps: float32 19 us, 5.3 TB/s, the rate of a large copy, float64
// 41, 4.9; 5 padded prompts x 777 x 1001 (single elements, see conv_vectors), 3 taps: 8.
template <typename T, int K, int VW>
__global__ void __launch_bounds__(256) conv_fwd_kernel(ConvArgs a) {
  constexpr int U = kConvUnroll;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t c = id % a.cv * VW, bs = id / a.cv, b = bs / a.nseg, s = bs % a.nseg;
  if (b >= a.B) return;
  const int64_t len = seq_len(a.lengths, b, a.T);
  const int64_t t0 = s * a.seg, t1 = t0 + a.seg < a.T ? t0 + a.seg : a.T;
  const T* xb = (const T*)a.x + b * a.sx.b + c;
  T* yb = (T*)a.y + b * a.sy.b + c;
  T w[K][VW], bias[VW], win[K - 1 + U][VW];
#pragma unroll
  for (int k = 0; k < K; ++k) vload<T, VW>(w[k], (const T*)a.w + k * a.C + c);
  if (a.b) {
    vload<T, VW>(bias, (const T*)a.b + c);
  } else {
#pragma unroll
    for (int e = 0; e < VW; ++e) bias[e] = T(0);
  }
#pragma unroll
  for (int j = 0; j < K - 1; ++j) conv_row<T, K, VW>(win[j], a, xb, b, t0 - (K - 1) + j, len, c);
  for (int64_t t = t0; t < t1; t += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) conv_row<T, K, VW>(win[K - 1 + u], a, xb, b, t + u, len, c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      T y[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        T p = bias[e];
#pragma unroll
        for (int k = 0; k < K; ++k) p = fma(w[k][e], win[u + k][e], p);
        y[e] = t + u >= len ? T(0) : a.silu ? p * sigmoid(p) : p;
      }
      if (t + u < t1) vstore<T, VW>(yb + (t + u) * a.sy.t, y);
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int e = 0; e < VW; ++e) win[j][e] = win[U + j][e];
  }
  // the last K - 1 inputs, by the segment that holds the sequence's end
  const int64_t last = len > 0 ? len - 1 : 0;
  if (a.state_out && last >= t0 && last < t1)
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      T r[VW];
      conv_row<T, K, VW>(r, a, xb, b, len - (K - 1) + j, len, c);
      vstore<T, VW>((T*)a.state_out + (b * (K - 1) + j) * a.C + c, r);
    }
}

// Backward of a segment: g'[t] = g[t] act'(pre[t]) for the segment's positions
// and the K - 1 after it, dx[t] = sum_k w[k] g'[t + K - 1 - k], and the
// segment's own terms of dw[k] = sum_t g'[t] x[t - K + 1 + k] and db = sum_t g'[t],
// summed over segments in a fixed order by a second kernel. The first segment
// also owns the positions of the state. 8 x 1024 x 1536, 4 taps: float32 32 us,
// 4.7 TB/s, and 4 for the sums; float64 99, 3.1 TB/s (a float64 exponential per element).
template <typename T, int K, int VW>
__global__ void __launch_bounds__(256) conv_bwd_kernel(ConvArgs a) {
  constexpr int U = kConvUnroll;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t c = id % a.cv * VW, bs = id / a.cv, b = bs / a.nseg, s = bs % a.nseg;
  if (b >= a.B) return;
  const int64_t len = seq_len(a.lengths, b, a.T);
  const int64_t t0 = s * a.seg, t1 = t0 + a.seg < a.T ? t0 + a.seg : a.T;
  const T* xb = (const T*)a.x + b * a.sx.b + c;
  const T* gb = (const T*)a.g + b * a.sg.b + c;
  T* dxb = (T*)a.dx + b * a.sdx.b + c;
  T w[K][VW], bias[VW], win[K - 1 + U][VW], gp[K - 1 + U][VW], dw[K][VW], db[VW];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    vload<T, VW>(w[k], (const T*)a.w + k * a.C + c);
#pragma unroll
    for (int e = 0; e < VW; ++e) dw[k][e] = T(0);
  }
  if (a.b) {
    vload<T, VW>(bias, (const T*)a.b + c);
  } else {
#pragma unroll
    for (int e = 0; e < VW; ++e) bias[e] = T(0);
  }
#pragma unroll
  for (int e = 0; e < VW; ++e) db[e] = T(0);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) {
    conv_row<T, K, VW>(win[j], a, xb, b, t0 - (K - 1) + j, len, c);
#pragma unroll
    for (int e = 0; e < VW; ++e) gp[j][e] = T(0);
  }
  // gp[j] is g'[t - (K - 1) + j]; position t gives dx[t - (K - 1)]
  const int64_t tend = t1 + K - 1;
  for (int64_t t = t0; t < tend; t += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      conv_row<T, K, VW>(win[K - 1 + u], a, xb, b, t + u, len, c);
      if (t + u < len) {
        vload<T, VW>(gp[K - 1 + u], gb + (t + u) * a.sg.t);
      } else {
#pragma unroll
        for (int e = 0; e < VW; ++e) gp[K - 1 + u][e] = T(0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = t + u < len, mine = t + u < t1 && in;
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        T g = gp[K - 1 + u][e];
        if (a.silu) {
          T p = bias[e];
#pragma unroll
          for (int k = 0; k < K; ++k) p = fma(w[k][e], win[u + k][e], p);
          const T sg = sigmoid(p);
          g = g * (sg * fma(p, T(1) - sg, T(1)));
          if (!in) g = T(0);
          gp[K - 1 + u][e] = g;
        }
        if (mine) {
          db[e] = db[e] + g;
#pragma unroll
          for (int k = 0; k < K; ++k) dw[k][e] = fma(g, win[u + k][e], dw[k][e]);
        }
      }
      const int64_t at = t + u - (K - 1);
      T d[VW];
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        T v = T(0);
#pragma unroll
        for (int k = 0; k < K; ++k) v = fma(w[k][e], gp[u + K - 1 - k][e], v);
        d[e] = v;
      }
      if (at < t1) {
        if (at >= t0) {
          vstore<T, VW>(dxb + at * a.sdx.t, d);
        } else if (at < 0 && a.dstate) {
          vstore<T, VW>((T*)a.dstate + (b * (K - 1) + (K - 1 + at)) * a.C + c, d);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < K - 1; ++j)
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        win[j][e] = win[U + j][e];
        gp[j][e] = gp[U + j][e];
      }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) vstore<T, VW>((T*)a.parts + (bs * (K + 1) + k) * a.C + c, dw[k]);
  vstore<T, VW>((T*)a.parts + (bs * (K + 1) + K) * a.C + c, db);
}

// dw [K, C] and db [C] (NULL: not wanted): the segments' terms [parts][K + 1][C].
// A block sums 64 columns, each of its 16 waves every 16th part with eight
// loads in flight, then the waves' sums in order.
template <typename T>
__global__ void __launch_bounds__(1024) conv_sum_kernel(const T* __restrict__ parts, int64_t n, int64_t KC, int64_t C,
                                                        T* __restrict__ dw, T* __restrict__ db) {
  __shared__ T sh[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t cols = KC + C, c = (int64_t)blockIdx.x * 64 + lane;
  T s = T(0);
  if (c < cols) {
    int64_t p = w;
    for (; p + 16 * 7 < n; p += 128) {
      T v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = parts[(p + 16 * u) * cols + c];
#pragma unroll
      for (int u = 0; u < 8; ++u) s = s + v[u];
    }
    for (; p < n; p += 16) s = s + parts[p * cols + c];
  }
  sh[w][lane] = s;
  __syncthreads();
  if (w != 0 || c >= cols) return;
  s = T(0);
#pragma unroll
  for (int v = 0; v < 16; ++v) s = s + sh[v][lane];
  if (c < KC)
    dw[c] = s;
  else if (db)
    db[c - KC] = s;
}

// One position per sequence: the state's K - 1 rows and the new input give y,
// and the state moves on by one row in place: a launch (4 x 256, 4 taps: 2.1 us;
// 512 x 1536: 5.7, float64 8.2).
template <typename T, int K, int VW>
__global__ void __launch_bounds__(256) conv_step_kernel(ConvArgs a) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t c = id % a.cv * VW, b = id / a.cv;
  if (b >= a.B) return;
  T win[K][VW], y[VW];
  T* st = (T*)a.state_out + b * (K - 1) * a.C + c;
#pragma unroll
  for (int j = 0; j < K - 1; ++j) vload<T, VW>(win[j], st + j * a.C);
  vload<T, VW>(win[K - 1], (const T*)a.x + b * a.sx.b + c);
  if (a.b) {
    vload<T, VW>(y, (const T*)a.b + c);
  } else {
#pragma unroll
    for (int e = 0; e < VW; ++e) y[e] = T(0);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    T w[VW];
    vload<T, VW>(w, (const T*)a.w + k * a.C + c);
#pragma unroll
    for (int e = 0; e < VW; ++e) y[e] = fma(w[e], win[k][e], y[e]);
  }
#pragma unroll
  for (int e = 0; e < VW; ++e) y[e] = a.silu ? y[e] * sigmoid(y[e]) : y[e];
  vstore<T, VW>((T*)a.y + b * a.sy.b + c, y);
#pragma unroll
  for (int j = 0; j < K - 1; ++j) vstore<T, VW>(st + j * a.C, win[j + 1]);
}

enum ConvOp { CONV_FWD, CONV_BWD, CONV_STEP };

template <typename T, int K, int VW>
static void conv_launch(ConvOp op, const ConvArgs& a, unsigned grid) {
  if (op == CONV_FWD) conv_fwd_kernel<T, K, VW><<<grid, 256, 0, stream()>>>(a);
  if (op == CONV_BWD) conv_bwd_kernel<T, K, VW><<<grid, 256, 0, stream()>>>(a);
  if (op == CONV_STEP) conv_step_kernel<T, K, VW><<<grid, 256, 0, stream()>>>(a);
}

template <typename T, int VW>
static void conv_taps(ConvOp op, const ConvArgs& a, int K, unsigned grid) {
  switch (K) {
    case 1: return conv_launch<T, 1, VW>(op, a, grid);
    case 2: return conv_launch<T, 2, VW>(op, a, grid);
    case 3: return conv_launch<T, 3, VW>(op, a, grid);
    case 4: return conv_launch<T, 4, VW>(op, a, grid);
    case 5: return conv_launch<T, 5, VW>(op, a, grid);
    case 6: return conv_launch<T, 6, VW>(op, a, grid);
    case 7: return conv_launch<T, 7, VW>(op, a, grid);
    default: return conv_launch<T, 8, VW>(op, a, grid);
  }
}

// Vectors of channels per row: whole 16-byte ones where every row is aligned to
// them, as the vector type asks, else single elements. (The hardware asks for a
// dword's alignment only: vectors for the bulk of such rows remain to be built.)
template <typename T>
static void conv_vectors(ConvArgs& a) {
  constexpr int VW = 16 / sizeof(T);
  const void* ptrs[] = {a.y, a.state_out, a.dx, a.dstate, a.x, a.w, a.b, a.state, a.g};
  const int64_t steps[] = {a.C, a.sx.b, a.sx.t, a.sy.b, a.sy.t, a.sg.b, a.sg.t, a.sdx.b, a.sdx.t};
  bool vec = true;
  for (const void* p : ptrs) vec = vec && aligned(p, 16);
  for (int64_t s : steps) vec = vec && s % VW == 0;
  a.cv = vec ? a.C / VW : a.C;
}

// Positions per thread: the longest segments that leave 600 threads per CU.
// 8 x 1024 x 1536 float32, forward / backward in us: 8 positions (1536 threads
// per CU) 20.2 / 40.4, 16: 18.7 / 32.1, 32: 22.8 / 35.0, 64: 36.8 / 52.6; short
// segments load more rows twice and leave more terms of dw to sum.
static void conv_segments(ConvArgs& a) {
  a.seg = 64;
  while (a.seg > 8 && a.B * cdiv(a.T, a.seg) * a.cv < (int64_t)num_cus() * 600) a.seg /= 2;
  a.nseg = cdiv(a.T, a.seg);
}

// rows: threads per vector of channels.
template <typename T>
static int conv_run(ConvOp op, const ConvArgs& a, int K, int64_t rows, const char* what) {
  const int64_t blocks = cdiv(a.cv * rows, 256);
  DTMI_CHECK(blocks <= 0x7fffffff, "%s: too many elements", what);
  if (a.cv != a.C)
    conv_taps<T, 16 / sizeof(T)>(op, a, K, (unsigned)blocks);
  else
    conv_taps<T, 1>(op, a, K, (unsigned)blocks);
  LAUNCH_CHECK(what);
  return DTMI_OK;
}

template <typename T>
static int conv_fwd(ConvArgs& a, int K) {
  conv_vectors<T>(a);
  conv_segments(a);
  return conv_run<T>(CONV_FWD, a, K, a.B * a.nseg, "dtmi_conv_fwd");
}
template <typename T>
static int conv_step(ConvArgs& a, int K) {
  conv_vectors<T>(a);
  return conv_run<T>(CONV_STEP, a, K, a.B, "dtmi_conv_step");
}

static int conv_shape(const char* what, int dtype, int64_t B, int64_t T, int64_t C, int64_t K) {
  DTMI_CHECK(dtype == DTMI_F32 || dtype == DTMI_F64, "%s: dtype must be DTMI_F32 or DTMI_F64 (got %d)", what, dtype);
  DTMI_CHECK(B >= 0 && T >= 0 && C >= 0, "%s: negative size", what);
  DTMI_CHECK(K >= 1 && K <= 8, "%s: 1 to 8 taps (got %lld)", what, (long long)K);
  return DTMI_OK;
}

}  // namespace dtmi

using namespace dtmi;

DTMI_EXPORT int dtmi_conv_fwd(int dtype, int64_t B, int64_t T, int64_t C, int64_t K, const void* x,
                              const int64_t* x_strides, const void* w, const void* b, const void* state,
                              const int64_t* lengths, int silu, void* y, const int64_t* y_strides, void* state_out) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  if (int rc = conv_shape("dtmi_conv_fwd", dtype, B, T, C, K)) return rc;
  if (B == 0 || C == 0) return DTMI_OK;
  DTMI_CHECK(w && (T == 0 || (x && y && x_strides && y_strides)), "dtmi_conv_fwd: NULL operand");
  if (T == 0) {  // the state passes through
    if (!state_out || K == 1) return DTMI_OK;
    const size_t bytes = (size_t)B * (K - 1) * C * (dtype == DTMI_F32 ? 4 : 8);
    return state ? dtmi_memcpy_d2d(state_out, state, bytes) : dtmi_zero_bytes(state_out, bytes);
  }
  ConvArgs a{};
  a.y = y, a.state_out = state_out, a.x = x, a.w = w, a.b = b, a.state = state, a.lengths = lengths;
  a.sx = {x_strides[0], x_strides[1]}, a.sy = {y_strides[0], y_strides[1]};
  a.B = B, a.T = T, a.C = C, a.silu = silu;
  TimedLaunch tl(DTMI_FAM_OTHER, 2.0 * B * T * C * (dtype == DTMI_F32 ? 4 : 8));
  return dtype == DTMI_F32 ? conv_fwd<float>(a, (int)K) : conv_fwd<double>(a, (int)K);
  DTMI_BODY_END
}

template <typename T>
static int conv_bwd(ConvArgs& a, int K, void* dw, void* db) {
  conv_vectors<T>(a);
  conv_segments(a);
  const int64_t parts = a.B * a.nseg;
  DTMI_CHECK(parts <= 0x7fffffff, "dtmi_conv_bwd: too many elements");
  void* p = nullptr;
  if (int rc = pool_alloc(&p, (size_t)parts * (K + 1) * a.C * sizeof(T))) return rc;
  a.parts = p;
  int rc = conv_run<T>(CONV_BWD, a, K, parts, "dtmi_conv_bwd");
  if (rc == DTMI_OK) {
    conv_sum_kernel<T><<<(unsigned)cdiv((K + 1) * a.C, 64), 1024, 0, stream()>>>((const T*)p, parts, K * a.C, a.C, (T*)dw,
                                                                               (T*)db);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) rc = fail_hip(e, "dtmi_conv_bwd", __FILE__, __LINE__);
  }
  pool_free(p);
  return rc;
}

DTMI_EXPORT int dtmi_conv_bwd(int dtype, int64_t B, int64_t T, int64_t C, int64_t K, const void* x,
                              const int64_t* x_strides, const void* w, const void* b, const void* state,
                              const int64_t* lengths, int silu, const void* g, const int64_t* g_strides, void* dx,
                              const int64_t* dx_strides, void* dw, void* db, void* dstate) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  if (int rc = conv_shape("dtmi_conv_bwd", dtype, B, T, C, K)) return rc;
  if (C == 0) return DTMI_OK;
  const size_t es = dtype == DTMI_F32 ? 4 : 8;
  DTMI_CHECK(w && dw, "dtmi_conv_bwd: NULL operand");
  if (B == 0 || T == 0) {
    int rc = dtmi_zero_bytes(dw, (size_t)K * C * es);
    if (rc == DTMI_OK && db) rc = dtmi_zero_bytes(db, (size_t)C * es);
    if (rc == DTMI_OK && dstate && B * (K - 1) > 0) rc = dtmi_zero_bytes(dstate, (size_t)B * (K - 1) * C * es);
    return rc;
  }
  DTMI_CHECK(x && g && dx && x_strides && g_strides && dx_strides, "dtmi_conv_bwd: NULL operand");
  ConvArgs a{};
  a.x = x, a.w = w, a.b = b, a.state = state, a.g = g, a.lengths = lengths, a.dx = dx, a.dstate = dstate;
  a.sx = {x_strides[0], x_strides[1]}, a.sg = {g_strides[0], g_strides[1]}, a.sdx = {dx_strides[0], dx_strides[1]};
  a.B = B, a.T = T, a.C = C, a.silu = silu;
  TimedLaunch tl(DTMI_FAM_OTHER, 3.0 * B * T * C * es);
  return dtype == DTMI_F32 ? conv_bwd<float>(a, (int)K, dw, db) : conv_bwd<double>(a, (int)K, dw, db);
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_conv_step(int dtype, int64_t B, int64_t C, int64_t K, const void* x, int64_t x_stride,
                               const void* w, const void* b, void* state, int silu, void* y, int64_t y_stride) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  if (int rc = conv_shape("dtmi_conv_step", dtype, B, 1, C, K)) return rc;
  if (B == 0 || C == 0) return DTMI_OK;
  DTMI_CHECK(x && w && y && (state || K == 1), "dtmi_conv_step: NULL operand");
  ConvArgs a{};
  a.x = x, a.w = w, a.b = b, a.state_out = state, a.y = y;
  a.sx.b = x_stride, a.sy.b = y_stride;
  a.B = B, a.C = C, a.silu = silu;
  TimedLaunch tl(DTMI_FAM_OTHER, 2.0 * B * C * K * (dtype == DTMI_F32 ? 4 : 8));
  return dtype == DTMI_F32 ? conv_step<float>(a, (int)K) : conv_step<double>(a, (int)K);
  DTMI_BODY_END
}
