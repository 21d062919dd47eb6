// Selective state space scan over [B, T, C] activations: every channel c keeps
// N states that decay at a rate the input chooses,
//   d[t, c]    = softplus(dt[t, c] + bias[c])          (or dt + bias)
//   h[t, c, n] = exp(d[t, c] A[c, n]) h[t-1, c, n] + d[t, c] u[t, c] B[t, g, n]
//   y[t, c]    = sum_n C[t, g, n] h[t, c, n] + D[c] u[t, c]
//   out        = y silu(z)                              (or y)
// with B and C shared by the channels of a group g. Positions at and past a
// sequence's length do nothing: their outputs and gradients are zero and
// the state stays.
//
// Mapping. A lane owns a channel, a wave 64 channels and 4 of their states,
// a block as many waves as cover the states (N up to 64: 16 waves); the
// recurrence runs in registers over tiles of TT positions. The waves of a
// block share what does not depend on the state: each stages its rows of a
// tile (softplus, d u, the gate) in LDS for all, and the per-wave sums over
// states are added through LDS in wave order. So the exponentials and
// products per state, which bound the kernel (one quarter-rate v_exp_f32 and
// four full-rate instructions per state and step), are all that is repeated.
//
// Parallelism over T. B * C / 64 blocks fill the card in training; a long
// prompt of few channels does not. Its positions are split into segments: one
// pass finds each segment's end state from a zero start and its sum of d, a
// small kernel chains the segments (the decay over a segment is
// exp(A sum d): no products of decays are kept), and the full pass starts
// each segment from its true state. Results do not depend on timing; the
// number of segments follows from the shape alone.
#include "seqmath.h"

namespace dtmi {

constexpr int kStates = 4;  // states per lane
constexpr double kLog2e = 1.4426950408889634;

// Positions per tile; the state before each tile is kept for the backward.
template <typename T>
__host__ __device__ constexpr int tile_len() {
  return sizeof(T) == 4 ? 16 : 8;
}
// Positions whose per-wave sums pass through LDS together in the forward.
template <typename T>
__host__ __device__ constexpr int sum_len(int W) {
  const int n = (sizeof(T) == 4 ? 64 : 32) / W, t = tile_len<T>();
  return n < t ? n : t;
}
// Positions whose states and decays a backward wave holds in registers at a
// time (8 per position and lane): a whole tile's would leave room for one wave
// per SIMD, so a tile is gone over in parts, the states before each part
// rebuilt once. Sixteen waves share the registers of a block of twice the size.
template <typename T>
__host__ __device__ constexpr int held_len(int W) {
  return (sizeof(T) == 4 ? 8 : 4) / (W <= 8 ? 1 : 2);
}
static int waves_for(int64_t N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// Element strides of the batch axis and of positions (below 2^31, checked on the host).
struct Rows {
  int64_t b;
  int t;
};

struct ScanArgs {
  const void *u, *dt, *A, *Bm, *Cm, *D, *z, *bias, *h0, *g;
  const int64_t* lengths;
  void *out, *hT, *kept;
  void *du, *ddt, *dz, *dh0;
  void *dBp, *dCp;      // [channel tiles of a group][B][T][G][N], contiguous
  void *prm;            // [B * segments][N + 2][C]: dA, dD, dbias terms
  void *carry, *dsum;   // [B][segments][N][C], [B][segments][C]
  Rows su, sdt, sz, sout, sg, sdu, sddt, sdz, sB, sC;
  int64_t gB, gC;       // group strides of B and C
  int64_t B, T, C, N, G;
  int seglen;           // positions per segment, a multiple of the tile
  int nseg, ct, tpg;    // segments; channel tiles in all and per group
  int softplus;
};

struct ScanBlock {
  int64_t b, c, c0;    // c0: the wave's first channel
  unsigned at;         // the lane's channel from c0 on (an idle lane: the group's last)
  int len, lo, hi;     // the sequence's length, the segment's positions
  int seg, grp, tile;  // segment, group, channel tile within the group
  bool on;
};

__device__ __forceinline__ ScanBlock scan_block(const ScanArgs& a) {
  ScanBlock k;
  const unsigned id = blockIdx.x, bs = id / (unsigned)a.ct, ct = id - bs * (unsigned)a.ct;
  k.b = bs / (unsigned)a.nseg;
  k.seg = (int)(bs % (unsigned)a.nseg);
  k.grp = (int)(ct / (unsigned)a.tpg);
  k.tile = (int)(ct % (unsigned)a.tpg);
  const int64_t each = a.C / a.G, off = (int64_t)k.tile * 64 + (threadIdx.x & 63);
  k.on = off < each;
  k.c = k.grp * each + off;
  k.c0 = k.grp * each + (int64_t)k.tile * 64;
  k.at = (unsigned)(k.on ? off : each - 1) - (unsigned)k.tile * 64u;
  k.len = (int)seq_len(a.lengths, k.b, a.T);
  k.lo = k.seg * a.seglen;
  k.hi = (int)(a.T - k.lo > a.seglen ? k.lo + a.seglen : a.T);
  return k;
}

template <typename T>
__device__ __forceinline__ T step_size(T raw, int softp) {
  return softp ? softplus(raw) : raw;
}

// A wave's rows of a tile (r = w, w + W, ...) and the block's share of the
// tile's maps, on their way from global memory. Positions at and past the
// length read the last one that holds data and are masked when the tile is
// staged, so no load waits for a branch.
template <typename T, int W, int TT>
struct Tile {
  static constexpr int RPW = (TT + W - 1) / W, NP = W * kStates, MAPS = (TT * NP + 64 * W - 1) / (64 * W);
  T u[RPW], d[RPW], z[RPW], g[RPW], b[MAPS], c[MAPS];
  // p: the wave's first channel, so row addresses are scalars and a lane adds 32 bits
  __device__ __forceinline__ void rows(T (&x)[RPW], const T* __restrict__ p, int st, int t0, int len, int w, unsigned at) {
    if (t0 + (TT > W ? TT : W) <= len) {
      const T* q = p + (int64_t)(t0 + w) * st;
#pragma unroll
      for (int i = 0; i < RPW; ++i, q += (int64_t)W * st) x[i] = q[at];
    } else {
#pragma unroll
      for (int i = 0; i < RPW; ++i) {
        const int t = t0 + w + W * i;
        x[i] = (p + (int64_t)(t < len ? t : len - 1) * st)[at];
      }
    }
  }
  __device__ __forceinline__ void map(T (&x)[MAPS], const T* __restrict__ p, int st, int t0, int len, int N) {
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      const int f = threadIdx.x + 64 * W * i, n = f % NP, t = t0 + f / NP;
      x[i] = p[(int64_t)(t < len ? t : len - 1) * st + (n < N ? n : N - 1)];
    }
  }
  static __device__ __forceinline__ void put_map(T* __restrict__ s, const T (&x)[MAPS], int t0, int len, int N) {
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      const int f = threadIdx.x + 64 * W * i;
      if (TT * NP % (64 * W) != 0 && f >= TT * NP) continue;
      s[f] = t0 + f / NP < len && f % NP < N ? x[i] : T(0);
    }
  }
};

// CARRY: only the segment's end state from a zero start, and its sum of d.
template <typename T, int W, bool CARRY>
__global__ void __launch_bounds__(64 * W) scan_fwd_kernel(ScanArgs a) {
  constexpr int NS = kStates, TT = tile_len<T>(), YT = sum_len<T>(W);
  using In = Tile<T, W, TT>;
  constexpr int RPW = In::RPW, NP = In::NP;
  __shared__ __attribute__((aligned(16))) T sB[TT * NP], sC[CARRY ? 1 : TT * NP];
  __shared__ T sd[TT][64], sx[TT][64], yp[CARRY ? 1 : W][CARRY ? 1 : YT][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ScanBlock k = scan_block(a);
  const int N = (int)a.N, n0 = w * NS;
  const T* up = (const T*)a.u + k.b * a.su.b + k.c0;
  const T* dp = (const T*)a.dt + k.b * a.sdt.b + k.c0;
  const T* zp = a.z ? (const T*)a.z + k.b * a.sz.b + k.c0 : nullptr;
  const T* Bp = (const T*)a.Bm + k.b * a.sB.b + k.grp * a.gB;
  const T* Cp = (const T*)a.Cm + k.b * a.sC.b + k.grp * a.gC;
  T* op = CARRY ? nullptr : (T*)a.out + k.b * a.sout.b + k.c0;
  const T bias = a.bias ? ((const T*)a.bias + k.c0)[k.at] : T(0);
  const T Dc = !CARRY && a.D ? ((const T*)a.D + k.c0)[k.at] : T(0);
  T A2[NS], h[NS], total = T(0);
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    A2[j] = n0 + j < N ? ((const T*)a.A)[(k.c0 + k.at) * N + n0 + j] * T(kLog2e) : T(0);
    h[j] = T(0);
    if (!CARRY && n0 + j < N) {
      if (a.nseg > 1)
        h[j] = ((const T*)a.carry)[((k.b * a.nseg + k.seg) * N + n0 + j) * a.C + k.c0 + k.at];
      else if (a.h0)
        h[j] = ((const T*)a.h0)[(k.b * a.C + k.c0 + k.at) * N + n0 + j];
    }
  }
  const int64_t ntiles = (a.T + TT - 1) / TT;
  const int stop = k.hi < k.len ? k.hi : k.len;  // positions at and past it do nothing
  In in;
  auto fetch = [&](int t0) {
    in.rows(in.u, up, a.su.t, t0, k.len, w, k.at);
    in.rows(in.d, dp, a.sdt.t, t0, k.len, w, k.at);
    in.map(in.b, Bp, a.sB.t, t0, k.len, N);
    if constexpr (!CARRY) in.map(in.c, Cp, a.sC.t, t0, k.len, N);
    if constexpr (!CARRY) {
      if (zp) in.rows(in.z, zp, a.sz.t, t0, k.len, w, k.at);
    }
  };
  if (k.lo < stop) fetch(k.lo);
  for (int t0 = k.lo; t0 < stop; t0 += TT) {
    T ur[RPW], zr[RPW];
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = w + W * i;
      if (W * RPW != TT && r >= TT) break;
      const bool on = t0 + r < k.len;
      const T d = on ? step_size(in.d[i] + bias, a.softplus) : T(0);
      ur[i] = on ? in.u[i] : T(0);
      if (!CARRY) zr[i] = in.z[i];
      sd[r][lane] = d;
      sx[r][lane] = d * ur[i];
    }
    In::put_map(sB, in.b, t0, k.len, N);
    if constexpr (!CARRY) In::put_map(sC, in.c, t0, k.len, N);
    if constexpr (!CARRY) {
      if (a.kept && k.on) {
        T* kp = (T*)a.kept + ((k.b * ntiles + t0 / TT) * N + n0) * a.C + k.c0;
#pragma unroll
        for (int j = 0; j < NS; ++j)
          if (n0 + j < N) (kp + j * a.C)[k.at] = h[j];
      }
    }
    __syncthreads();
    if (t0 + TT < stop) fetch(t0 + TT);
#pragma unroll
    for (int s = 0; s < TT / YT; ++s) {
#pragma unroll
      for (int q = 0; q < YT; ++q) {
        const int r = s * YT + q;
        const T d = sd[r][lane], x = sx[r][lane];
        T y = T(0);
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          h[j] = fma(exp2_of(d * A2[j]), h[j], x * sB[r * NP + n0 + j]);
          if constexpr (!CARRY) y = fma(sC[r * NP + n0 + j], h[j], y);
        }
        if constexpr (CARRY)
          total = total + d;
        else
          yp[w][q][lane] = y;
      }
      __syncthreads();
      if constexpr (!CARRY) {
        T* q = op + (int64_t)(t0 + w) * a.sout.t;
#pragma unroll
        for (int i = 0; i < RPW; ++i, q += (int64_t)W * a.sout.t) {
          const int r = w + W * i;
          if (r / YT != s || r >= TT) continue;
          T y = T(0);
#pragma unroll
          for (int v = 0; v < W; ++v) y = y + yp[v][r % YT][lane];
          y = fma(Dc, ur[i], y);
          if (zp) y = y * (zr[i] * sigmoid(zr[i]));
          if (k.on && t0 + r < stop) q[k.at] = y;
        }
        if (TT != YT) __syncthreads();
      }
    }
  }
  if (!k.on) return;
  if constexpr (CARRY) {
    const int64_t at = k.b * a.nseg + k.seg;
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (n0 + j < N) ((T*)a.carry)[(at * N + n0 + j) * a.C + k.c] = h[j];
    if (w == 0) ((T*)a.dsum)[at * a.C + k.c] = total;
  } else {
    for (int t = (stop > k.lo ? stop : k.lo) + w; t < k.hi; t += W) (op + (int64_t)t * a.sout.t)[k.at] = T(0);
    if (a.hT && k.seg == a.nseg - 1) {
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (n0 + j < N) ((T*)a.hT)[(k.b * a.C + k.c) * N + n0 + j] = h[j];
    }
  }
}

// Chains the segments in place: carry[s] becomes what enters segment s, in
// the order of time (forward: from h0) or against it (backward: from zero;
// what leaves the first segment is the gradient of h0).
template <typename T>
__global__ void __launch_bounds__(256) scan_chain_kernel(ScanArgs a, int backward) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t c = id % a.C, bn = id / a.C, n = bn % a.N, b = bn / a.N;
  if (b >= a.B) return;
  const T A2 = ((const T*)a.A)[c * a.N + n] * T(kLog2e);
  T in = !backward && a.h0 ? ((const T*)a.h0)[(b * a.C + c) * a.N + n] : T(0);
  // the loads do not wait for the chain: eight segments' at a time
  constexpr int U = 8;
  const int64_t step = backward ? -1 : 1, from = b * a.nseg + (backward ? a.nseg - 1 : 0);
  T* p = (T*)a.carry + (from * a.N + n) * a.C + c;
  const T* d = (const T*)a.dsum + from * a.C + c;
  for (int i = 0; i < a.nseg; i += U) {
    T local[U], sum[U];
#pragma unroll
    for (int v = 0; v < U; ++v) {
      const int64_t at = step * (i + v < a.nseg ? i + v : a.nseg - 1);
      local[v] = p[at * a.N * a.C];
      sum[v] = d[at * a.C];
    }
#pragma unroll
    for (int v = 0; v < U; ++v) {
      if (i + v >= a.nseg) break;
      p[step * (i + v) * a.N * a.C] = in;
      in = fma(exp2_of(A2 * sum[v]), in, local[v]);
    }
  }
}

// x of the lane that DPP control CTRL names
template <int CTRL>
__device__ __forceinline__ float lane_of(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double lane_of(double x) {
  typedef int i2 __attribute__((ext_vector_type(2)));
  i2 v = __builtin_bit_cast(i2, x);
  v.x = __builtin_amdgcn_update_dpp(0, v.x, CTRL, 0xf, 0xf, true);
  v.y = __builtin_amdgcn_update_dpp(0, v.y, CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, v);
}
// p's sums of lane halves (ROW = 32: lanes l and l + 32; 16: l and l + 16) in the
// lower half of each pair, q's in the upper: one exchange, one addition
template <int ROW>
__device__ __forceinline__ void swap_rows(unsigned& p, unsigned& q) {
  if constexpr (ROW == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(p, q, false, false);
    p = r[0], q = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane16_swap(p, q, false, false);
    p = r[0], q = r[1];
  }
}
template <int ROW>
__device__ __forceinline__ float fold(float p, float q) {
  unsigned a = __builtin_bit_cast(unsigned, p), b = __builtin_bit_cast(unsigned, q);
  swap_rows<ROW>(a, b);
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
template <int ROW>
__device__ __forceinline__ double fold(double p, double q) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  u2 a = __builtin_bit_cast(u2, p), b = __builtin_bit_cast(u2, q);
  unsigned ax = a.x, ay = a.y, bx = b.x, by = b.y;
  swap_rows<ROW>(ax, bx);
  swap_rows<ROW>(ay, by);
  a = u2{ax, ay}, b = u2{bx, by};
  return __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b);
}
// Sums over the wave of 8 values, 18 instructions: lane l ends with that of
// value l / 8. Each step halves the values a lane holds; the last three add
// within the eight lanes that hold the same one.
template <typename T>
__device__ __forceinline__ T sum8(const T (&v)[8], bool upper8) {
  const T x0 = fold<32>(v[0], v[4]), x1 = fold<32>(v[1], v[5]), x2 = fold<32>(v[2], v[6]), x3 = fold<32>(v[3], v[7]);
  const T y0 = fold<16>(x0, x2), y1 = fold<16>(x1, x3);
  T r = (upper8 ? y1 : y0) + lane_of<0x128>(upper8 ? y0 : y1);  // row_ror:8
  r = r + lane_of<0x141>(r);                                    // row_half_mirror
  r = r + lane_of<0xB1>(r);                                     // quad_perm 1,0,3,2
  return r + lane_of<0x4E>(r);                                  // quad_perm 2,3,0,1
}

// The backward over a segment, last tile first. dh carries the gradient of the
// state to the earlier positions:
//   dh += dy C[t];  dx = sum_n dh B[t];  q = dh exp(d A) h[t-1];  dh *= exp(d A)
//   du = d dx + D dy,  dd = sum_n A q + u dx,  dA += d q
//   dB[t] = sum_c dh d u,  dC[t] = sum_c dy h[t]
// A tile's states are rebuilt in registers from the state kept before it. The
// sums over a wave's channels (dB, dC) are taken as sum8, eight values of a
// step together, and eight steps' results leave a wave as one LDS write.
// CARRY: only dh over the segment, and its sum of d.
template <typename T, int W, bool CARRY>
__global__ void __launch_bounds__(64 * W, W <= 8 ? 2 : 4) scan_bwd_kernel(ScanArgs a) {
  constexpr int NS = kStates, TT = tile_len<T>(), HT = held_len<T>(W);
  using In = Tile<T, W, TT>;
  constexpr int RPW = In::RPW, NP = In::NP, RB = HT < 8 ? HT : 8;
  __shared__ T sd[TT][64], sx[CARRY ? 1 : TT][64], sy[TT][64], yp[CARRY ? 1 : 3][CARRY ? 1 : W][CARRY ? 1 : HT][64];
  __shared__ __attribute__((aligned(16))) T sB[CARRY ? 1 : TT * NP], sC[TT * NP];
  __shared__ T sg[CARRY ? 1 : TT][CARRY ? 1 : 2 * NP];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ScanBlock k = scan_block(a);
  const int N = (int)a.N, n0 = w * NS;
  const T* up = (const T*)a.u + k.b * a.su.b + k.c0;
  const T* dp = (const T*)a.dt + k.b * a.sdt.b + k.c0;
  const T* zp = a.z ? (const T*)a.z + k.b * a.sz.b + k.c0 : nullptr;
  const T* gp = (const T*)a.g + k.b * a.sg.b + k.c0;
  const T* Bp = (const T*)a.Bm + k.b * a.sB.b + k.grp * a.gB;
  const T* Cp = (const T*)a.Cm + k.b * a.sC.b + k.grp * a.gC;
  const T bias = a.bias ? ((const T*)a.bias + k.c0)[k.at] : T(0);
  const T Dc = a.D ? ((const T*)a.D + k.c0)[k.at] : T(0);
  T An[NS], A2[NS], dh[NS], dA[NS], total = T(0), dD = T(0), dbias = T(0);
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    An[j] = n0 + j < N ? ((const T*)a.A)[(k.c0 + k.at) * N + n0 + j] : T(0);
    A2[j] = An[j] * T(kLog2e);
    dA[j] = dh[j] = T(0);
    if (!CARRY && a.nseg > 1 && n0 + j < N)
      dh[j] = ((const T*)a.carry)[((k.b * a.nseg + k.seg) * N + n0 + j) * a.C + k.c0 + k.at];
  }
  const int64_t ntiles = (a.T + TT - 1) / TT;
  const int stop = k.hi < k.len ? k.hi : k.len;
  // this block's dB and dC terms: row t of part k.tile
  const int64_t prow = ((k.tile * a.B + k.b) * a.T) * a.G + k.grp;
  if constexpr (!CARRY) {  // positions past the sequence: zeros
    const int from = stop > k.lo ? stop : k.lo;
    if (k.on)
      for (int t = from + w; t < k.hi; t += W) {
        ((T*)a.du)[k.b * a.sdu.b + (int64_t)t * a.sdu.t + k.c] = T(0);
        ((T*)a.ddt)[k.b * a.sddt.b + (int64_t)t * a.sddt.t + k.c] = T(0);
        if (zp) ((T*)a.dz)[k.b * a.sdz.b + (int64_t)t * a.sdz.t + k.c] = T(0);
      }
    for (int64_t f = threadIdx.x; f < (int64_t)(k.hi - from) * N; f += 64 * W) {
      const int64_t at = (prow + (from + f / N) * a.G) * N + f % N;
      ((T*)a.dBp)[at] = T(0);
      ((T*)a.dCp)[at] = T(0);
    }
  }
  In in;
  T kept[NS];
  auto fetch = [&](int t0) {
    in.rows(in.d, dp, a.sdt.t, t0, k.len, w, k.at);
    in.rows(in.g, gp, a.sg.t, t0, k.len, w, k.at);
    if (zp) in.rows(in.z, zp, a.sz.t, t0, k.len, w, k.at);
    in.map(in.c, Cp, a.sC.t, t0, k.len, N);
    if constexpr (!CARRY) {
      in.rows(in.u, up, a.su.t, t0, k.len, w, k.at);
      in.map(in.b, Bp, a.sB.t, t0, k.len, N);
      const T* kp = (const T*)a.kept + ((k.b * ntiles + t0 / TT) * N + n0) * a.C + k.c0;
#pragma unroll
      for (int j = 0; j < NS; ++j) kept[j] = n0 + j < N ? (kp + j * a.C)[k.at] : T(0);
    }
  };
  const int first = k.lo + (stop - 1 - k.lo) / TT * TT;
  T *dup = nullptr, *ddp = nullptr, *dzp = nullptr;
  if constexpr (!CARRY) {
    dup = (T*)a.du + k.b * a.sdu.b + k.c0;
    ddp = (T*)a.ddt + k.b * a.sddt.b + k.c0;
    if (zp) dzp = (T*)a.dz + k.b * a.sdz.b + k.c0;
  }
  if (k.lo < stop) fetch(first);
  for (int t0 = first; k.lo < stop && t0 >= k.lo; t0 -= TT) {
    T ur[RPW], zr[RPW], gr[RPW], dr[RPW], rr[RPW];
    __syncthreads();  // the previous tile's LDS has been read
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = w + W * i;
      if (W * RPW != TT && r >= TT) break;
      const bool on = t0 + r < k.len && k.on;  // an idle lane's terms are zero
      rr[i] = in.d[i] + bias;
      gr[i] = on ? in.g[i] : T(0);
      dr[i] = on ? step_size(rr[i], a.softplus) : T(0);
      zr[i] = zp && on ? in.z[i] : T(0);
      const T dy = zp ? gr[i] * (zr[i] * sigmoid(zr[i])) : gr[i];
      sd[r][lane] = dr[i];
      sy[r][lane] = dy;
      if constexpr (!CARRY) {
        ur[i] = on ? in.u[i] : T(0);
        sx[r][lane] = dr[i] * ur[i];
      }
    }
    In::put_map(sC, in.c, t0, k.len, N);
    if constexpr (CARRY) {
      __syncthreads();
      if (t0 > k.lo) fetch(t0 - TT);
#pragma unroll
      for (int r = TT - 1; r >= 0; --r) {
        const T d = sd[r][lane], dy = sy[r][lane];
        total = total + d;
#pragma unroll
        for (int j = 0; j < NS; ++j) dh[j] = exp2_of(d * A2[j]) * fma(dy, sC[r * NP + n0 + j], dh[j]);
      }
    } else {
      In::put_map(sB, in.b, t0, k.len, N);
      // the states before each part of the tile
      T start[TT / HT][NS];
#pragma unroll
      for (int j = 0; j < NS; ++j) start[0][j] = kept[j];
      __syncthreads();
      if (t0 > k.lo) fetch(t0 - TT);
#pragma unroll
      for (int s = 1; s < TT / HT; ++s) {
#pragma unroll
        for (int j = 0; j < NS; ++j) start[s][j] = start[s - 1][j];
#pragma unroll
        for (int q = 0; q < HT; ++q) {
          const int r = (s - 1) * HT + q;
          const T d = sd[r][lane], x = sx[r][lane];
#pragma unroll
          for (int j = 0; j < NS; ++j)
            start[s][j] = fma(exp2_of(d * A2[j]), start[s][j], x * sB[r * NP + n0 + j]);
          if (q % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
      }
      T sums = T(0);
#pragma unroll
      for (int s = TT / HT - 1; s >= 0; --s) {
        T dec[HT][NS], h[HT + 1][NS];  // h[q]: the states before position q of the part
#pragma unroll
        for (int j = 0; j < NS; ++j) h[0][j] = start[s][j];
#pragma unroll
        for (int q = 0; q < HT; ++q) {
          const int r = s * HT + q;
          const T d = sd[r][lane], x = sx[r][lane];
#pragma unroll
          for (int j = 0; j < NS; ++j) {
            dec[q][j] = exp2_of(d * A2[j]);
            h[q + 1][j] = fma(dec[q][j], h[q][j], x * sB[r * NP + n0 + j]);
          }
          if (q % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int q = HT - 1; q >= 0; --q) {
          const int r = s * HT + q;
          const T d = sd[r][lane], x = sx[r][lane], dy = sy[r][lane];
          T dx = T(0), e = T(0), y = T(0), v[8];
#pragma unroll
          for (int j = 0; j < NS; ++j) {
            const T Cn = sC[r * NP + n0 + j], Bn = sB[r * NP + n0 + j];
            y = fma(Cn, h[q + 1][j], y);
            v[4 + j] = dy * h[q + 1][j];
            dh[j] = fma(dy, Cn, dh[j]);
            dx = fma(dh[j], Bn, dx);
            v[j] = dh[j] * x;
            dh[j] = dh[j] * dec[q][j];
            const T p = dh[j] * h[q][j];
            e = fma(An[j], p, e);
            dA[j] = fma(d, p, dA[j]);
          }
          yp[0][w][q][lane] = y;
          yp[1][w][q][lane] = dx;
          yp[2][w][q][lane] = e;
          // lane l keeps value l / 8 of step r with r % 8 = l % 8
          const T sum = sum8<T>(v, lane & 8);
          sums = (lane & (RB - 1)) == r % RB ? sum : sums;
          __builtin_amdgcn_sched_barrier(0);
          if (r % RB == 0 && (lane & 7) < RB)
            sg[r + (lane & 7)][(lane >> 5) * NP + n0 + ((lane >> 3) & 3)] = sums;
        }
        __syncthreads();
        T *qu = dup + (int64_t)(t0 + w) * a.sdu.t, *qd = ddp + (int64_t)(t0 + w) * a.sddt.t;
        T* qz = dzp + (int64_t)(t0 + w) * a.sdz.t;
#pragma unroll
        for (int i = 0; i < RPW; ++i, qu += (int64_t)W * a.sdu.t, qd += (int64_t)W * a.sddt.t, qz += (int64_t)W * a.sdz.t) {
          const int r = w + W * i;
          if (r / HT != s || r >= TT) continue;
          T y = T(0), dx = T(0), e = T(0);
#pragma unroll
          for (int v = 0; v < W; ++v) {
            y = y + yp[0][v][r % HT][lane];
            dx = dx + yp[1][v][r % HT][lane];
            e = e + yp[2][v][r % HT][lane];
          }
          const bool put = k.on && t0 + r < stop;
          T dy = gr[i];
          if (zp) {
            const T sz = sigmoid(zr[i]);
            y = fma(Dc, ur[i], y);
            const T dz = gr[i] * y * (sz * fma(zr[i], T(1) - sz, T(1)));
            dy = gr[i] * (zr[i] * sz);
            if (put) qz[k.at] = dz;
          }
          T dd = fma(dx, ur[i], e);
          if (a.softplus) dd = dd * sigmoid(rr[i]);
          if (put) {
            dD = fma(dy, ur[i], dD);
            dbias = dbias + dd;
            qu[k.at] = fma(dx, dr[i], Dc * dy);
            qd[k.at] = dd;
          }
        }
        if (s > 0) __syncthreads();
      }
      const int rows = (int)(stop - t0 < TT ? stop - t0 : TT);
      for (int f = threadIdx.x; f < rows * NP; f += 64 * W) {
        const int r = f / NP, n = f % NP;
        if (n >= N) continue;
        const int64_t at = (prow + (t0 + r) * a.G) * N + n;
        ((T*)a.dBp)[at] = sg[r][n];
        ((T*)a.dCp)[at] = sg[r][NP + n];
      }
    }
  }
  if constexpr (CARRY) {
    if (!k.on) return;
    const int64_t at = k.b * a.nseg + k.seg;
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (n0 + j < N) ((T*)a.carry)[(at * N + n0 + j) * a.C + k.c] = dh[j];
    if (w == 0) ((T*)a.dsum)[at * a.C + k.c] = total;
  } else {
    // D's and the bias's terms lie with the waves that own the rows
    __syncthreads();
    yp[0][w][0][lane] = dD;
    yp[1][w][0][lane] = dbias;
    __syncthreads();
    if (!k.on) return;
    T* prm = (T*)a.prm + (k.b * a.nseg + k.seg) * (N + 2) * a.C + k.c;
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (n0 + j < N) {
        prm[(n0 + j) * a.C] = dA[j];
        if (a.dh0 && k.seg == 0) ((T*)a.dh0)[(k.b * a.C + k.c) * N + n0 + j] = dh[j];
      }
    if (w == 0) {
      dD = dbias = T(0);
#pragma unroll
      for (int v = 0; v < W; ++v) {
        dD = dD + yp[0][v][0][lane];
        dbias = dbias + yp[1][v][0][lane];
      }
      prm[N * a.C] = dD;
      prm[(N + 1) * a.C] = dbias;
    }
  }
}

// dA [C, N], dD [C] and dbias [C] (NULL: not wanted): the blocks' terms in order
template <typename T>
__global__ void __launch_bounds__(256) scan_param_kernel(const T* __restrict__ prm, int64_t parts, int64_t N, int64_t C,
                                                         T* __restrict__ dA, T* __restrict__ dD, T* __restrict__ dbias) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (N + 2) * C) return;
  const int64_t n = id / C, c = id % C;
  T s = T(0);
  for (int64_t p = 0; p < parts; ++p) s = s + prm[p * (N + 2) * C + id];
  if (n < N)
    dA[c * N + n] = s;
  else if (n == N && dD)
    dD[c] = s;
  else if (n == N + 1 && dbias)
    dbias[c] = s;
}

// dB and dC: the channel tiles' terms in order, into their own layouts
template <typename T>
__global__ void __launch_bounds__(256) scan_map_kernel(ScanArgs a, T* __restrict__ dB, BT sB, int64_t gB,
                                                       T* __restrict__ dC, BT sC, int64_t gC) {
  const int64_t n1 = a.B * a.T * a.G * a.N, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= n1) return;
  const int64_t n = id % a.N, row = id / a.N, g = row % a.G, bt = row / a.G, t = bt % a.T, b = bt / a.T;
  T x = T(0), y = T(0);
  for (int p = 0; p < a.tpg; ++p) {
    x = x + ((const T*)a.dBp)[p * n1 + id];
    y = y + ((const T*)a.dCp)[p * n1 + id];
  }
  dB[b * sB.b + t * sB.t + g * gB + n] = x;
  dC[b * sC.b + t * sC.t + g * gC + n] = y;
}

// One position per sequence, the states in place. A group of LPC lanes owns a
// channel, four states each; bound by reading and writing the states once.
template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(256) scan_step_kernel(ScanArgs a) {
  constexpr int NS = kStates;
  typedef T vt __attribute__((ext_vector_type(4)));
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t bc = id / LPC, c = bc % a.C, b = bc / a.C;
  const int n0 = (int)(id % LPC) * NS, N = (int)a.N;
  const bool on = b < a.B;
  T y = T(0);
  T u = T(0);
  if (on) {
    u = ((const T*)a.u)[b * a.su.b + c];
    T raw = ((const T*)a.dt)[b * a.sdt.b + c];
    if (a.bias) raw = raw + ((const T*)a.bias)[c];
    const T d = step_size(raw, a.softplus), x = d * u;
    const int64_t g = c / (a.C / a.G);
    const T* Bp = (const T*)a.Bm + b * a.sB.b + g * a.gB + n0;
    const T* Cp = (const T*)a.Cm + b * a.sC.b + g * a.gC + n0;
    const T* Ap = (const T*)a.A + c * N + n0;
    T* hp = (T*)a.hT + (b * a.C + c) * N + n0;
    if constexpr (VEC) {
      if (n0 < N) {
        const vt A = *(const vt*)Ap;
        vt h = *(const vt*)hp;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          h[j] = fma(exp2_of(d * (A[j] * T(kLog2e))), h[j], x * Bp[j]);
          y = fma(Cp[j], h[j], y);
        }
        *(vt*)hp = h;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (n0 + j < N) {
          const T h = fma(exp2_of(d * (Ap[j] * T(kLog2e))), hp[j], x * Bp[j]);
          hp[j] = h;
          y = fma(Cp[j], h, y);
        }
    }
  }
#pragma unroll
  for (int m = 1; m < LPC; m <<= 1) y = y + __shfl_xor(y, m, 64);
  if (!on || n0 != 0) return;
  if (a.D) y = fma(((const T*)a.D)[c], u, y);
  if (a.z) {
    const T z = ((const T*)a.z)[b * a.sz.b + c];
    y = y * (z * sigmoid(z));
  }
  ((T*)a.out)[b * a.sout.b + c] = y;
}

template <typename T, bool BWD, bool CARRY>
static void scan_launch(const ScanArgs& a, int W) {
  const unsigned grid = (unsigned)(a.B * a.nseg * a.ct);
#define SCAN_W(w)                                                                  \
  case w:                                                                          \
    if constexpr (BWD)                                                             \
      scan_bwd_kernel<T, w, CARRY><<<grid, 64 * w, 0, stream()>>>(a);              \
    else                                                                           \
      scan_fwd_kernel<T, w, CARRY><<<grid, 64 * w, 0, stream()>>>(a);              \
    break;
  switch (W) {
    SCAN_W(1) SCAN_W(2) SCAN_W(4) SCAN_W(8) SCAN_W(16)
  }
#undef SCAN_W
}

static int scan_tile(int dtype) {
  return dtype == DTMI_F32 ? tile_len<float>() : tile_len<double>();
}

// Segments of T: one where B * C / 64 blocks already occupy the card. A split
// costs the exponentials a second time, so it has to more than double the
// blocks that run at once; then enough segments for two blocks per CU, of at
// least two tiles each.
static void scan_segments(ScanArgs& a, int TT, int per_cu) {
  const int64_t blocks = a.B * a.ct, want = per_cu * (int64_t)num_cus(), tiles = cdiv(a.T, TT);
  int64_t s = blocks >= num_cus() ? 1 : want / blocks;
  if (s > tiles / 2) s = tiles / 2;
  if (s < 1) s = 1;
  a.seglen = (int)(cdiv(tiles, s) * TT);
  a.nseg = (int)cdiv(a.T, a.seglen);
}

static int scan_shape(const char* what, int dtype, int64_t B, int64_t T, int64_t C, int64_t N, int64_t G) {
  DTMI_CHECK(dtype == DTMI_F32 || dtype == DTMI_F64, "%s: dtype must be DTMI_F32 or DTMI_F64 (got %d)", what, dtype);
  DTMI_CHECK(B >= 0 && T >= 0 && C >= 0, "%s: negative size", what);
  DTMI_CHECK(T <= 0x7fffff00, "%s: too many positions", what);
  DTMI_CHECK(N >= 1 && N <= 64, "%s: 1 to 64 states (got %lld)", what, (long long)N);
  DTMI_CHECK(G >= 1 && C % G == 0, "%s: %lld channels do not form %lld groups", what, (long long)C, (long long)G);
  return DTMI_OK;
}

template <typename T>
static int scan_chain(ScanArgs& a, int W, bool backward) {
  if (backward)
    scan_launch<T, true, true>(a, W);
  else
    scan_launch<T, false, true>(a, W);
  LAUNCH_CHECK("scan: segment pass");
  scan_chain_kernel<T><<<(unsigned)cdiv(a.B * a.N * a.C, 256), 256, 0, stream()>>>(a, backward ? 1 : 0);
  LAUNCH_CHECK("scan: segment chain");
  return DTMI_OK;
}

template <typename T>
static int scan_fwd(ScanArgs& a) {
  const int W = waves_for(a.N);
  scan_segments(a, tile_len<T>(), 4);
  DTMI_CHECK(a.B * a.nseg * a.ct <= 0x7fffffff && a.B * a.N * a.C <= (int64_t)0x7fffffff * 256,
             "dtmi_scan_fwd: too many elements");
  void* ws = nullptr;
  int rc = DTMI_OK;
  if (a.nseg > 1) {
    const size_t n = (size_t)a.B * a.nseg * a.C;
    rc = pool_alloc(&ws, n * (a.N + 1) * sizeof(T));
    if (rc) return rc;
    a.carry = ws;
    a.dsum = (T*)ws + n * a.N;
    rc = scan_chain<T>(a, W, false);
  }
  if (rc == DTMI_OK) {
    scan_launch<T, false, false>(a, W);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) rc = fail_hip(e, "dtmi_scan_fwd", __FILE__, __LINE__);
  }
  if (ws) pool_free(ws);
  return rc;
}

template <typename T>
static int scan_bwd(ScanArgs& a, void* dA, void* dB, BT sdB, int64_t gdB, void* dC, BT sdC, int64_t gdC, void* dD,
                    void* dbias) {
  const int W = waves_for(a.N);
  scan_segments(a, tile_len<T>(), 2);
  const int64_t maps = a.B * a.T * a.G * a.N;
  DTMI_CHECK(a.B * a.nseg * a.ct <= 0x7fffffff && a.B * a.N * a.C <= (int64_t)0x7fffffff * 256 &&
                 maps <= (int64_t)0x7fffffff * 256,
             "dtmi_scan_bwd: too many elements");
  // dB and dC terms per channel tile, parameter terms per block row, and the
  // segments' carries
  const size_t np = (size_t)a.tpg * maps, nprm = (size_t)a.B * a.nseg * (a.N + 2) * a.C;
  const size_t nc = a.nseg > 1 ? (size_t)a.B * a.nseg * (a.N + 1) * a.C : 0;
  void* ws = nullptr;
  if (int rc = pool_alloc(&ws, (2 * np + nprm + nc) * sizeof(T))) return rc;
  a.dBp = ws;
  a.dCp = (T*)ws + np;
  a.prm = (T*)ws + 2 * np;
  int rc = DTMI_OK;
  if (a.nseg > 1) {
    a.carry = (T*)ws + 2 * np + nprm;
    a.dsum = (T*)a.carry + (size_t)a.B * a.nseg * a.N * a.C;
    rc = scan_chain<T>(a, W, true);
  }
  if (rc == DTMI_OK) {
    scan_launch<T, true, false>(a, W);
    scan_param_kernel<T><<<(unsigned)cdiv((a.N + 2) * a.C, 256), 256, 0, stream()>>>(
        (const T*)a.prm, a.B * a.nseg, a.N, a.C, (T*)dA, (T*)dD, (T*)dbias);
    scan_map_kernel<T><<<(unsigned)cdiv(maps, 256), 256, 0, stream()>>>(a, (T*)dB, sdB, gdB, (T*)dC, sdC, gdC);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) rc = fail_hip(e, "dtmi_scan_bwd", __FILE__, __LINE__);
  }
  pool_free(ws);
  return rc;
}

static BT bt(const int64_t* s) { return s ? BT{s[0], s[1]} : BT{0, 0}; }
// False for a distance between positions that 32 bits do not hold.
static bool rows_of(Rows& r, const int64_t* s) {
  if (!s) return true;
  r = {s[0], (int)s[1]};
  return s[1] == r.t;
}

static void scan_tiles(ScanArgs& a) {
  a.tpg = (int)cdiv(a.C / a.G, 64);
  a.ct = (int)(a.tpg * a.G);
}

}  // namespace dtmi

using namespace dtmi;

DTMI_EXPORT int dtmi_scan_kept(int dtype, int64_t B, int64_t T, int64_t C, int64_t N, int64_t* count) {
  DTMI_BODY_BEGIN
  if (int rc = scan_shape("dtmi_scan_kept", dtype, B, T, C, N, 1)) return rc;
  DTMI_CHECK(count, "dtmi_scan_kept: NULL result");
  *count = B * cdiv(T, scan_tile(dtype)) * N * C;
  return DTMI_OK;
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_scan_fwd(int dtype, int64_t B, int64_t T, int64_t C, int64_t N, int64_t G, const void* u,
                              const int64_t* u_strides, const void* dt, const int64_t* dt_strides, const void* A,
                              const void* Bm, const int64_t* B_strides, const void* Cm, const int64_t* C_strides,
                              const void* D, const void* z, const int64_t* z_strides, const void* dt_bias,
                              const void* state, const int64_t* lengths, int softplus, void* out,
                              const int64_t* out_strides, void* state_out, void* kept) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  if (int rc = scan_shape("dtmi_scan_fwd", dtype, B, T, C, N, G)) return rc;
  if (B == 0 || C == 0) return DTMI_OK;
  if (T == 0) {
    if (!state_out) return DTMI_OK;
    const size_t bytes = (size_t)B * C * N * (dtype == DTMI_F32 ? 4 : 8);
    return state ? dtmi_memcpy_d2d(state_out, state, bytes) : dtmi_zero_bytes(state_out, bytes);
  }
  DTMI_CHECK(u && dt && A && Bm && Cm && out && u_strides && dt_strides && B_strides && C_strides && out_strides &&
                 (!z || z_strides),
             "dtmi_scan_fwd: NULL operand");
  ScanArgs a{};
  a.u = u, a.dt = dt, a.A = A, a.Bm = Bm, a.Cm = Cm, a.D = D, a.z = z, a.bias = dt_bias, a.h0 = state;
  a.lengths = lengths, a.out = out, a.hT = state_out, a.kept = kept, a.softplus = softplus;
  DTMI_CHECK(rows_of(a.su, u_strides) && rows_of(a.sdt, dt_strides) && rows_of(a.sz, z_strides) &&
                 rows_of(a.sout, out_strides) && rows_of(a.sB, B_strides) && rows_of(a.sC, C_strides),
             "dtmi_scan_fwd: positions more than 2^31 elements apart");
  a.gB = B_strides[2], a.gC = C_strides[2];
  a.B = B, a.T = T, a.C = C, a.N = N, a.G = G;
  scan_tiles(a);
  TimedLaunch tl(DTMI_FAM_OTHER, 7.0 * B * T * C * N);
  return dtype == DTMI_F32 ? scan_fwd<float>(a) : scan_fwd<double>(a);
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_scan_bwd(int dtype, int64_t B, int64_t T, int64_t C, int64_t N, int64_t G, const void* u,
                              const int64_t* u_strides, const void* dt, const int64_t* dt_strides, const void* A,
                              const void* Bm, const int64_t* B_strides, const void* Cm, const int64_t* C_strides,
                              const void* D, const void* z, const int64_t* z_strides, const void* dt_bias,
                              const int64_t* lengths, int softplus, const void* kept, const void* g,
                              const int64_t* g_strides, void* du, const int64_t* du_strides, void* ddt,
                              const int64_t* ddt_strides, void* dA, void* dB, const int64_t* dB_strides, void* dC,
                              const int64_t* dC_strides, void* dD, void* dz, const int64_t* dz_strides, void* ddt_bias,
                              void* dstate) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  if (int rc = scan_shape("dtmi_scan_bwd", dtype, B, T, C, N, G)) return rc;
  if (C == 0) return DTMI_OK;
  const size_t es = dtype == DTMI_F32 ? 4 : 8;
  DTMI_CHECK(dA, "dtmi_scan_bwd: NULL operand");
  if (B == 0 || T == 0) {
    int rc = dtmi_zero_bytes(dA, (size_t)C * N * es);
    if (rc == DTMI_OK && dD) rc = dtmi_zero_bytes(dD, (size_t)C * es);
    if (rc == DTMI_OK && ddt_bias) rc = dtmi_zero_bytes(ddt_bias, (size_t)C * es);
    if (rc == DTMI_OK && dstate && B > 0) rc = dtmi_zero_bytes(dstate, (size_t)B * C * N * es);
    return rc;
  }
  DTMI_CHECK(u && dt && A && Bm && Cm && kept && g && du && ddt && dB && dC && u_strides && dt_strides && B_strides &&
                 C_strides && g_strides && du_strides && ddt_strides && dB_strides && dC_strides &&
                 (!z || (z_strides && dz && dz_strides)),
             "dtmi_scan_bwd: NULL operand");
  ScanArgs a{};
  a.u = u, a.dt = dt, a.A = A, a.Bm = Bm, a.Cm = Cm, a.D = D, a.z = z, a.bias = dt_bias, a.g = g;
  a.lengths = lengths, a.kept = const_cast<void*>(kept), a.softplus = softplus;
  a.du = du, a.ddt = ddt, a.dz = dz, a.dh0 = dstate;
  DTMI_CHECK(rows_of(a.su, u_strides) && rows_of(a.sdt, dt_strides) && rows_of(a.sz, z_strides) &&
                 rows_of(a.sg, g_strides) && rows_of(a.sB, B_strides) && rows_of(a.sC, C_strides) &&
                 rows_of(a.sdu, du_strides) && rows_of(a.sddt, ddt_strides) && rows_of(a.sdz, dz_strides),
             "dtmi_scan_bwd: positions more than 2^31 elements apart");
  a.gB = B_strides[2], a.gC = C_strides[2];
  a.B = B, a.T = T, a.C = C, a.N = N, a.G = G;
  scan_tiles(a);
  TimedLaunch tl(DTMI_FAM_OTHER, 14.0 * B * T * C * N);
  const BT sdB = bt(dB_strides), sdC = bt(dC_strides);
  return dtype == DTMI_F32 ? scan_bwd<float>(a, dA, dB, sdB, dB_strides[2], dC, sdC, dC_strides[2], dD, ddt_bias)
                           : scan_bwd<double>(a, dA, dB, sdB, dB_strides[2], dC, sdC, dC_strides[2], dD, ddt_bias);
  DTMI_BODY_END
}

template <typename T>
static void scan_step(const ScanArgs& a) {
  const int lpc = waves_for(a.N);  // lanes per channel: the same 4-state slices
  const unsigned grid = (unsigned)cdiv(a.B * a.C * lpc, 256);
  const bool vec = a.N % 4 == 0 && aligned(a.A, 4 * sizeof(T)) && aligned(a.hT, 4 * sizeof(T));
#define STEP_L(l)                                                            \
  case l:                                                                    \
    if (vec)                                                                 \
      scan_step_kernel<T, l, true><<<grid, 256, 0, stream()>>>(a);           \
    else                                                                     \
      scan_step_kernel<T, l, false><<<grid, 256, 0, stream()>>>(a);          \
    break;
  switch (lpc) {
    STEP_L(1) STEP_L(2) STEP_L(4) STEP_L(8) STEP_L(16)
  }
#undef STEP_L
}

DTMI_EXPORT int dtmi_scan_step(int dtype, int64_t B, int64_t C, int64_t N, int64_t G, const void* u, int64_t u_stride,
                               const void* dt, int64_t dt_stride, const void* A, const void* Bm,
                               const int64_t* B_strides, const void* Cm, const int64_t* C_strides, const void* D,
                               const void* z, int64_t z_stride, const void* dt_bias, void* state, int softplus,
                               void* out, int64_t out_stride) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  if (int rc = scan_shape("dtmi_scan_step", dtype, B, 1, C, N, G)) return rc;
  if (B == 0 || C == 0) return DTMI_OK;
  DTMI_CHECK(u && dt && A && Bm && Cm && state && out && B_strides && C_strides, "dtmi_scan_step: NULL operand");
  DTMI_CHECK(B * C <= ((int64_t)1 << 34), "dtmi_scan_step: too many elements");
  ScanArgs a{};
  a.u = u, a.dt = dt, a.A = A, a.Bm = Bm, a.Cm = Cm, a.D = D, a.z = z, a.bias = dt_bias, a.hT = state, a.out = out;
  a.su.b = u_stride, a.sdt.b = dt_stride, a.sz.b = z_stride, a.sout.b = out_stride;
  a.sB.b = B_strides[0], a.gB = B_strides[1], a.sC.b = C_strides[0], a.gC = C_strides[1];
  a.B = B, a.C = C, a.N = N, a.G = G, a.softplus = softplus;
  TimedLaunch tl(DTMI_FAM_OTHER, 7.0 * B * C * N);
  if (dtype == DTMI_F32)
    scan_step<float>(a);
  else
    scan_step<double>(a);
  LAUNCH_CHECK("dtmi_scan_step");
  return DTMI_OK;
  DTMI_BODY_END
}
