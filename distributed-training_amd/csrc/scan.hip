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
// products per state, which bound the kernel (a v_exp_f32 of two issue slots and
// four instructions per state and step), are all that is repeated.
//
// Parallelism over T. B * C / 64 blocks fill the card in training; a long
// prompt of few channels does not. Its positions are split into segments: one
// pass finds each segment's end state from a zero start and its sum of d, a
// small kernel chains the segments (the decay over a segment is
// exp(A sum d): no products of decays are kept), and the full pass starts
// each segment from its true state. Results do not depend on timing; the
// number of segments follows from the shape alone.
#include "bufrsrc.h"
#include "seqmath.h"

namespace dtmi {

constexpr int kStates = 4;  // states per lane
constexpr double kLog2e = 1.4426950408889634, kLn2 = 0.6931471805599453;

// A in base 2, at least the type's lowest value: an A of -inf (-exp(log rate), when
// it overflows) forgets a state at once, but not where the step is 0
template <typename T>
__device__ __forceinline__ T decay_rate(T a) {
  constexpr T lowest = sizeof(T) == 4 ? T(-3.40282347e38f) : T(-1.7976931348623157e308);
  const T x = a * T(kLog2e);
  return x < lowest ? lowest : x;
}

// Positions per tile. The backward's sixteen waves have 128 registers a lane, which
// hold half a float32 tile (4 x 1024 x 1536 x 64: 16 positions spill, 732 us, 8: 472).
template <typename T>
__host__ __device__ constexpr int tile_len(int W, bool bwd) {
  return sizeof(T) == 4 && !(bwd && W == 16) ? 16 : 8;
}
// Positions whose per-wave sums pass through LDS together in the forward.
template <typename T>
__host__ __device__ constexpr int sum_len(int W) {
  const int n = (sizeof(T) == 4 ? 64 : 32) / W, t = tile_len<T>(W, false);
  return n < t ? n : t;
}
// Positions whose states and decays a backward wave holds in registers at a
// time (8 values per position and lane): a whole tile's would leave room for
// one wave per SIMD, so a tile is gone over in parts. Sixteen waves share the
// registers of a block of twice the size.
template <typename T>
__host__ __device__ constexpr int held_len(int W) {
  return (sizeof(T) == 4 ? 8 : 4) / (W <= 8 ? 1 : 2);
}
// Waves per SIMD the backward's registers are cut to: two of 219 (float32, 9 to
// 16 states; three of 168 spill, and a spill's store counts as one to wait for), one
// in float64 up to 16 states and for up to 4 states (a wave then stages all of a
// tile), where two spill. A block of eight waves is two per SIMD and one of sixteen
// four, whatever they need: float64 keeps 32 and 164 of a lane's values in memory there.
template <typename T>
__host__ __device__ constexpr int bwd_waves(int W) {
  return W == 16 ? 4 : W == 8 ? 2 : sizeof(T) == 4 && W > 1 ? 2 : 1;
}
// Positions per state kept for the backward, which rebuilds the states in
// between (16 states: two activations' memory). One per float32 part: at one per
// 16 positions 5 us less traffic and 10 us more of exponentials at 4 x 1024 x 1536 x
// 16. One per tile of eight where a part is shorter: there memory counts for more.
constexpr int kKeep = 8;
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
  int nseg, ct, tpg;    // segments; channel tiles in all and per group (a step: channels per group)
  int softplus;
};

struct ScanBlock {
  int64_t b, c, c0;    // the lane's channel, the first of the block's
  int len, lo, hi;     // the sequence's length, the segment's positions
  int seg, grp, tile;  // segment, group, channel tile within the group
  int cnt;             // channels of the block: lanes from there on are idle
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
  k.cnt = (int)(each - (int64_t)k.tile * 64 < 64 ? each - (int64_t)k.tile * 64 : 64);
  k.len = (int)seq_len(a.lengths, k.b, a.T);
  k.lo = k.seg * a.seglen;
  k.hi = (int)(a.T - k.lo > a.seglen ? k.lo + a.seglen : a.T);
  return k;
}

// d of one position, 0 where there is none. Both branches are the same for all
// lanes; the sum is formed ahead of them, so that they hold no wait for a load
// (the count of stores since would be lost, see Row).
template <typename T>
__device__ __forceinline__ T step_size(T raw, int softp, bool there) {
  asm volatile("" : "+v"(raw));
  const T d = softp ? softplus(raw) : raw;
  return there ? d : T(0);
}

template <typename T>
__device__ __forceinline__ void store_at(Rsrc r, int off, T x) {
  typedef int i2 __attribute__((ext_vector_type(2)));
  if constexpr (sizeof(T) == 4)
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, x), r, off, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(i2, x), r, off, 0, 0);
}

// A row of a block's channels (p: its first, the same for all lanes): a buffer
// that ends with the block's channels, or is empty for a row that is not there.
// Lanes and rows outside read 0 and write nothing. The addresses take no vector
// registers (64-bit lane addresses of a tile's rows in seven arrays took 56),
// and the tile loop's loads and stores no branches: where a store may or may
// not have been issued, the wait for the next tile's loads becomes a wait for
// every store as well, 1.7 us per tile for a wave alone on its SIMD.
template <typename T>
struct Row {
  Rsrc r;
  __device__ __forceinline__ Row(const T* p, bool there, int cnt) : r(make_rsrc(p, there ? cnt * (int)sizeof(T) : 0)) {}
  __device__ __forceinline__ T get() const {
    const int off = (threadIdx.x & 63) * (int)sizeof(T);
    if constexpr (sizeof(T) == 4)
      return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
    else
      return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
  }
  __device__ __forceinline__ void put(T x) const { store_at(r, (threadIdx.x & 63) * (int)sizeof(T), x); }
};

// A value the compiler takes as new: row addresses formed from it are computed
// where they are used, not carried as a scalar per row and array through the
// loop (more than the scalar registers hold).
__device__ __forceinline__ int renewed(int x) {
  asm volatile("" : "+s"(x));
  return x;
}

// s_waitcnt vmcnt(0) ahead of the tile loop: with loads in flight at its entry
// the first wait inside would cover both ways into the loop, which is every
// store of the tile before.
__device__ __forceinline__ void drain_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// A wave's rows of a tile (r = w, w + W, ...) and the block's share of the
// tile's maps, on their way from global memory.
template <typename T, int W, int TT>
struct Tile {
  static constexpr int RPW = (TT + W - 1) / W, NP = W * kStates, MAPS = (TT * NP + 64 * W - 1) / (64 * W);
  T u[RPW], d[RPW], z[RPW], g[RPW], b[MAPS], c[MAPS];
  __device__ __forceinline__ void rows(T (&x)[RPW], const T* __restrict__ p, int st, int t0, const ScanBlock& k, int w,
                                       bool there = true) {
    const T* q = p + (int64_t)(t0 + w) * st;
#pragma unroll
    for (int i = 0; i < RPW; ++i, q += (int64_t)W * st)
      x[i] = Row<T>(q, there && (unsigned)(t0 + w + W * i) < (unsigned)k.len, k.cnt).get();
  }
  // (a map's position outside the sequence reads one inside and is masked when staged)
  __device__ __forceinline__ void map(T (&x)[MAPS], const T* __restrict__ p, int st, int t0, int len, int N) {
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      const int f = threadIdx.x + 64 * W * i, n = f % NP, t = t0 + f / NP < len ? t0 + f / NP : len - 1;
      x[i] = p[(int64_t)(t > 0 ? t : 0) * st + (n < N ? n : N - 1)];
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

// What a wave reads from LDS for one position. The next positions' are asked
// for before the current ones' arithmetic, and kept there by scheduling
// barriers: left to itself the compiler reads them right before their use, and
// a wave alone on its SIMD then waits out the LDS latency at every position.
template <typename T>
struct Step {
  T d, x, g, b[kStates], c[kStates];
};
// Not where many waves share a SIMD's registers: there they cover each other's reads
// and the positions ahead would spill (4 x 1024 x 1536, us with and without: backward
// of 64 states 826 / 732 in float32, 3285 / 3015 in float64, of 32 in float64 1041 /
// 890; small, the forward and the segments' passes: 64 states in float64 1516 / 912).
template <typename T>
constexpr bool reads_ahead(int W, bool small) {
  return sizeof(T) == 4 ? small || W < 16 : W < (small ? 16 : 8);
}

// 4 x 1024 x 1536 x 16 float32: 100.7 M states and steps at 6 issue slots are 15
// us of vector instructions, the bytes 19; measured 36, and 25 for CARRY: the
// vector unit is busy for 77 % of the cycles (the stores of a tile, the sums over
// waves and the staging are the rest). Maps as scalar loads: 68 against 39 then.
// float64: 130 and 99, the library's exponential.
// CARRY: only the segment's end state from a zero start, and its sum of d.
template <typename T, int W, bool CARRY>
__global__ void __launch_bounds__(64 * W) scan_fwd_kernel(ScanArgs a) {
  constexpr int NS = kStates, TT = tile_len<T>(W, false), YT = sum_len<T>(W), KT = kKeep;
  using In = Tile<T, W, TT>;
  constexpr int RPW = In::RPW, NP = In::NP;
  constexpr bool AHEAD = reads_ahead<T>(W, true);
  __shared__ __attribute__((aligned(16))) T sB[TT * NP], sC[CARRY ? 1 : TT * NP];
  __shared__ T sd[TT][64], sx[TT][64], yp[CARRY ? 1 : W][CARRY ? 1 : YT][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ScanBlock k = scan_block(a);
  const int N = (int)a.N, n0 = w * NS;
  const T* up = (const T*)a.u + k.b * a.su.b + k.c0;
  const T* dp = (const T*)a.dt + k.b * a.sdt.b + k.c0;
  const T* zp = (const T*)a.z + k.b * a.sz.b + k.c0;
  const bool gate = a.z != nullptr, keep = a.kept != nullptr;
  const T* Bp = (const T*)a.Bm + k.b * a.sB.b + k.grp * a.gB;
  const T* Cp = (const T*)a.Cm + k.b * a.sC.b + k.grp * a.gC;
  T* op = CARRY ? nullptr : (T*)a.out + k.b * a.sout.b + k.c0;
  const T bias = a.bias ? Row<T>((const T*)a.bias + k.c0, true, k.cnt).get() : T(0);
  const T Dc = !CARRY && a.D ? Row<T>((const T*)a.D + k.c0, true, k.cnt).get() : T(0);
  T A2[NS], h[NS], total = T(0);
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    A2[j] = k.on && n0 + j < N ? decay_rate(((const T*)a.A)[k.c * N + n0 + j]) : T(0);
    h[j] = T(0);
    if (!CARRY && k.on && n0 + j < N) {
      if (a.nseg > 1)
        h[j] = ((const T*)a.carry)[((k.b * a.nseg + k.seg) * N + n0 + j) * a.C + k.c];
      else if (a.h0)
        h[j] = ((const T*)a.h0)[(k.b * a.C + k.c) * N + n0 + j];
    }
  }
  const int64_t nkept = (a.T + KT - 1) / KT;
  const int stop = k.hi < k.len ? k.hi : k.len;  // positions at and past it do nothing
  In in;
  auto fetch = [&](int from) {
    const int t0 = renewed(from);
    in.rows(in.u, up, a.su.t, t0, k, w);
    in.rows(in.d, dp, a.sdt.t, t0, k, w);
    in.map(in.b, Bp, a.sB.t, t0, k.len, N);
    if constexpr (!CARRY) in.map(in.c, Cp, a.sC.t, t0, k.len, N);
    if constexpr (!CARRY) {
      in.rows(in.z, zp, a.sz.t, t0, k, w, gate);
    }
  };
  if (k.lo < stop) fetch(k.lo);
  drain_loads();
  for (int t0 = k.lo; t0 < stop; t0 += TT) {
    T ur[RPW], zr[RPW];
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = w + W * i;
      if (W * RPW != TT && r >= TT) break;
      const T d = step_size(in.d[i] + bias, a.softplus, t0 + r < k.len);
      ur[i] = in.u[i];
      if (!CARRY) zr[i] = in.z[i];
      sd[r][lane] = d;
      sx[r][lane] = d * ur[i];
    }
    In::put_map(sB, in.b, t0, k.len, N);
    if constexpr (!CARRY) In::put_map(sC, in.c, t0, k.len, N);
    __syncthreads();
    fetch(t0 + TT);
    constexpr int PF = AHEAD ? 2 : 1;  // positions read together
    Step<T> at[PF], next[PF];
    auto read = [&](Step<T>(&x)[PF], int r) {
#pragma unroll
      for (int i = 0; i < PF; ++i) {
        x[i].d = sd[r + i][lane];
        x[i].x = sx[r + i][lane];
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          x[i].b[j] = sB[(r + i) * NP + n0 + j];
          if constexpr (!CARRY) x[i].c[j] = sC[(r + i) * NP + n0 + j];
        }
      }
    };
    if (AHEAD) read(at, 0);
#pragma unroll
    for (int s = 0; s < TT / YT; ++s) {
#pragma unroll
      for (int q = 0; q < YT; q += PF) {
        if (!AHEAD)
          read(at, s * YT + q);
        else if (s * YT + q + PF < TT)
          read(next, s * YT + q + PF);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < PF; ++i) {
          const int r = s * YT + q + i;
          if constexpr (!CARRY) {
            if (r % KT == 0) {
              const int t = renewed(t0) + r;
              const T* kp = (const T*)a.kept + ((k.b * nkept + t / KT) * N + n0) * a.C + k.c0;
#pragma unroll
              for (int j = 0; j < NS; ++j) Row<T>(kp + j * a.C, keep && t < stop && n0 + j < N, k.cnt).put(h[j]);
            }
          }
          T y = T(0);
#pragma unroll
          for (int j = 0; j < NS; ++j) {
            h[j] = fma(exp2_of(at[i].d * A2[j]), h[j], at[i].x * at[i].b[j]);
            if constexpr (!CARRY) y = fma(at[i].c[j], h[j], y);
          }
          if constexpr (CARRY)
            total = total + at[i].d;
          else
            yp[w][q + i][lane] = y;
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < (AHEAD ? PF : 0); ++i) at[i] = next[i];
      }
      __syncthreads();
      if constexpr (!CARRY) {
        const int tn = renewed(t0);
#pragma unroll
        for (int i = 0; i < RPW; ++i) {
          const int r = w + W * i;
          if ((W <= YT ? W * i / YT : r / YT) != s || r >= TT) continue;
          T y = T(0);
#pragma unroll
          for (int v = 0; v < W; ++v) y = y + yp[v][r % YT][lane];
          y = fma(Dc, ur[i], y);
          y = gate ? y * (zr[i] * sigmoid(zr[i])) : y;
          Row<T>(op + (int64_t)(tn + r) * a.sout.t, tn + r < stop, k.cnt).put(y);
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
    for (int t = (stop > k.lo ? stop : k.lo) + w; t < k.hi; t += W)
      Row<T>(op + (int64_t)t * a.sout.t, true, k.cnt).put(T(0));
    if (a.hT && k.seg == a.nseg - 1) {
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (n0 + j < N) ((T*)a.hT)[(k.b * a.C + k.c) * N + n0 + j] = h[j];
    }
  }
}

// Chains the segments in place: carry[s] becomes what enters segment s, in
// the order of time (forward: from h0) or against it (backward: from zero;
// what leaves the first segment is the gradient of h0). States that grow may do so
// beyond the type's range over a segment while their own value stays in it: 0 stays
// 0, and the growth is applied in two halves. Bound by the latency of
// its rounds of loads (64 segments of 1 x 768 x 16: 8.2 us).
template <typename T>
__global__ void __launch_bounds__(256) scan_chain_kernel(ScanArgs a, int backward) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t c = id % a.C, bn = id / a.C, n = bn % a.N, b = bn / a.N;
  if (b >= a.B) return;
  const T A2 = decay_rate(((const T*)a.A)[c * a.N + n]);
  T in = !backward && a.h0 ? ((const T*)a.h0)[(b * a.C + c) * a.N + n] : T(0);
  // the loads do not wait for the chain: sixteen segments' at a time
  constexpr int U = 16;
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
      const T half = exp2_of(T(.5) * A2 * sum[v]);
      in = in == T(0) ? local[v] : fma(in * half, half, local[v]);
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
// 4 x 1024 x 1536 x 16 float32: 100 us, and 27 for CARRY (float64 339 and 107). Per
// state and step 5 issue slots rebuild the state, 9 go back, 4.5 are the channel sums,
// beside the tile's staging; the vector unit is busy for 61 to 70 % of the cycles, two
// waves per SIMD leave its chains in view.
// CARRY: only dh over the segment, and its sum of d.
template <typename T, int W, bool CARRY>
__global__ void __launch_bounds__(64 * W, bwd_waves<T>(W)) scan_bwd_kernel(ScanArgs a) {
  constexpr int NS = kStates, TT = tile_len<T>(W, true), HT = held_len<T>(W), KT = kKeep;
  using In = Tile<T, W, TT>;
  constexpr int RPW = In::RPW, NP = In::NP, RB = HT < 8 ? HT : 8;
  constexpr bool AHEAD = reads_ahead<T>(W, CARRY);
  __shared__ T sd[TT][64], sx[CARRY ? 1 : TT][64], sy[TT][64], yp[CARRY ? 1 : 3][CARRY ? 1 : W][CARRY ? 1 : HT][64];
  __shared__ __attribute__((aligned(16))) T sB[CARRY ? 1 : TT * NP], sC[TT * NP];
  __shared__ T sg[CARRY ? 1 : TT][CARRY ? 1 : 2 * NP];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const ScanBlock k = scan_block(a);
  const int N = (int)a.N, n0 = w * NS;
  const T* up = (const T*)a.u + k.b * a.su.b + k.c0;
  const T* dp = (const T*)a.dt + k.b * a.sdt.b + k.c0;
  const T* zp = (const T*)a.z + k.b * a.sz.b + k.c0;
  const bool gate = a.z != nullptr;
  const T* gp = (const T*)a.g + k.b * a.sg.b + k.c0;
  const T* Bp = (const T*)a.Bm + k.b * a.sB.b + k.grp * a.gB;
  const T* Cp = (const T*)a.Cm + k.b * a.sC.b + k.grp * a.gC;
  const T bias = a.bias ? Row<T>((const T*)a.bias + k.c0, true, k.cnt).get() : T(0);
  const T Dc = a.D ? Row<T>((const T*)a.D + k.c0, true, k.cnt).get() : T(0);
  T A2[NS], dh[NS], dA[NS], total = T(0), dD = T(0), dbias = T(0);
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    A2[j] = k.on && n0 + j < N ? decay_rate(((const T*)a.A)[k.c * N + n0 + j]) : T(0);
    dA[j] = dh[j] = T(0);
    if (!CARRY && a.nseg > 1 && k.on && n0 + j < N)
      dh[j] = ((const T*)a.carry)[((k.b * a.nseg + k.seg) * N + n0 + j) * a.C + k.c];
  }
  const int64_t nkept = (a.T + KT - 1) / KT;
  const int stop = k.hi < k.len ? k.hi : k.len;
  // this block's dB and dC terms: row t of part k.tile
  const int64_t prow = ((k.tile * a.B + k.b) * a.T) * a.G + k.grp;
  if constexpr (!CARRY) {  // positions past the sequence: zeros
    const int from = stop > k.lo ? stop : k.lo;
    if (k.on)
      for (int t = from + w; t < k.hi; t += W) {
        ((T*)a.du)[k.b * a.sdu.b + (int64_t)t * a.sdu.t + k.c] = T(0);
        ((T*)a.ddt)[k.b * a.sddt.b + (int64_t)t * a.sddt.t + k.c] = T(0);
        if (gate) ((T*)a.dz)[k.b * a.sdz.b + (int64_t)t * a.sdz.t + k.c] = T(0);
      }
    for (int64_t f = threadIdx.x; f < (int64_t)(k.hi - from) * N; f += 64 * W) {
      const int64_t at = (prow + (from + f / N) * a.G) * N + f % N;
      ((T*)a.dBp)[at] = T(0);
      ((T*)a.dCp)[at] = T(0);
    }
  }
  In in;
  T kept[TT / KT][NS];
  auto fetch = [&](int from) {
    const int t0 = renewed(from);
    in.rows(in.d, dp, a.sdt.t, t0, k, w);
    in.rows(in.g, gp, a.sg.t, t0, k, w);
    in.rows(in.z, zp, a.sz.t, t0, k, w, gate);
    in.map(in.c, Cp, a.sC.t, t0, k.len, N);
    if constexpr (!CARRY) {
      in.rows(in.u, up, a.su.t, t0, k, w);
      in.map(in.b, Bp, a.sB.t, t0, k.len, N);
#pragma unroll
      for (int s = 0; s < TT / KT; ++s) {
        const int t = t0 + s * KT;
        const T* kp = (const T*)a.kept + ((k.b * nkept + t / KT) * N + n0) * a.C + k.c0;
#pragma unroll
        for (int j = 0; j < NS; ++j) kept[s][j] = Row<T>(kp + j * a.C, (unsigned)t < (unsigned)stop && n0 + j < N, k.cnt).get();
      }
    }
  };
  const int first = k.lo + (stop - 1 - k.lo) / TT * TT;
  T *dup = nullptr, *ddp = nullptr, *dzp = nullptr;
  if constexpr (!CARRY) {
    dup = (T*)a.du + k.b * a.sdu.b + k.c0;
    ddp = (T*)a.ddt + k.b * a.sddt.b + k.c0;
    dzp = (T*)a.dz + k.b * a.sdz.b + k.c0;
  }
  if (k.lo < stop) fetch(first);
  drain_loads();
  for (int t0 = first; k.lo < stop && t0 >= k.lo; t0 -= TT) {
    T ur[RPW], gz[RPW], ds[RPW];  // u; the factors of dz and ddt
    __syncthreads();  // the previous tile's LDS has been read
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int r = w + W * i;
      if (W * RPW != TT && r >= TT) break;
      // (of an idle lane or a position past the end u, g and z are zero, and so are all terms)
      const T raw = in.d[i] + bias, g = in.g[i];
      const T d = step_size(raw, a.softplus, t0 + r < k.len);
      const T z = in.z[i], sz = sigmoid(z), dy = gate ? g * (z * sz) : g;
      if constexpr (!CARRY) gz[i] = g * (sz * fma(z, T(1) - sz, T(1)));
      if constexpr (!CARRY) ds[i] = a.softplus ? sigmoid(raw) : T(1);
      sd[r][lane] = d;
      sy[r][lane] = dy;
      if constexpr (!CARRY) {
        ur[i] = in.u[i];
        sx[r][lane] = d * ur[i];
      }
    }
    In::put_map(sC, in.c, t0, k.len, N);
    if constexpr (CARRY) {
      __syncthreads();
      fetch(t0 - TT);
      constexpr int PF = AHEAD ? 2 : 1;  // positions read together
      Step<T> at[PF], next[PF];
      auto read = [&](Step<T>(&x)[PF], int r) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
          x[i].d = sd[r + i][lane];
          x[i].g = sy[r + i][lane];
#pragma unroll
          for (int j = 0; j < NS; ++j) x[i].c[j] = sC[(r + i) * NP + n0 + j];
        }
      };
      if (AHEAD) read(at, TT - PF);
#pragma unroll
      for (int r = TT - PF; r >= 0; r -= PF) {
        if (!AHEAD)
          read(at, r);
        else if (r > 0)
          read(next, r - PF);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = PF - 1; i >= 0; --i) {
          total = total + at[i].d;
#pragma unroll
          for (int j = 0; j < NS; ++j) dh[j] = exp2_of(at[i].d * A2[j]) * fma(at[i].g, at[i].c[j], dh[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < (AHEAD ? PF : 0); ++i) at[i] = next[i];
      }
    } else {
      In::put_map(sB, in.b, t0, k.len, N);
      // the states before each part of the tile
      T start[TT / HT][NS];
#pragma unroll
      for (int s = 0; s < TT / KT; ++s)
#pragma unroll
        for (int j = 0; j < NS; ++j) start[s * (KT / HT)][j] = kept[s][j];
      __syncthreads();
      fetch(t0 - TT);
      // those that were not kept
#pragma unroll
      for (int s = 1; s < TT / HT; ++s) {
        if (s % (KT / HT) == 0) continue;
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
        auto read = [&](int r, bool back) {
          Step<T> x;
          x.d = sd[r][lane];
          x.x = sx[r][lane];
          if (back) x.g = sy[r][lane];
#pragma unroll
          for (int j = 0; j < NS; ++j) {
            x.b[j] = sB[r * NP + n0 + j];
            if (back) x.c[j] = sC[r * NP + n0 + j];
          }
          return x;
        };
        Step<T> at;
        if (AHEAD) at = read(s * HT, false);
#pragma unroll
        for (int q = 0; q < HT; ++q) {
          Step<T> next;
          if (AHEAD)
            next = q + 1 < HT ? read(s * HT + q + 1, false) : read(s * HT + q, true);
          else
            at = read(s * HT + q, false);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < NS; ++j) {
            dec[q][j] = exp2_of(at.d * A2[j]);
            h[q + 1][j] = fma(dec[q][j], h[q][j], at.x * at.b[j]);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (AHEAD) at = next;
        }
#pragma unroll
        for (int q = HT - 1; q >= 0; --q) {
          const int r = s * HT + q;
          Step<T> next;
          if (AHEAD)
            next = q > 0 ? read(r - 1, true) : at;
          else
            at = read(r, true);
          __builtin_amdgcn_sched_barrier(0);
          T dx = T(0), e = T(0), y = T(0), v[8];
#pragma unroll
          for (int j = 0; j < NS; ++j) {
            y = fma(at.c[j], h[q + 1][j], y);
            v[4 + j] = at.g * h[q + 1][j];
            dh[j] = fma(at.g, at.c[j], dh[j]);
            dx = fma(dh[j], at.b[j], dx);
            v[j] = dh[j] * at.x;
            dh[j] = dh[j] * dec[q][j];
            const T p = dh[j] * h[q][j];
            e = fma(A2[j], p, e);
            dA[j] = fma(at.d, p, dA[j]);
          }
          if (AHEAD) at = next;
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
        const int tn = renewed(t0);
#pragma unroll
        for (int i = 0; i < RPW; ++i) {
          const int r = w + W * i;
          if ((W <= HT ? W * i / HT : r / HT) != s || r >= TT) continue;
          T y = T(0), dx = T(0), e = T(0);
#pragma unroll
          for (int v = 0; v < W; ++v) {
            y = y + yp[0][v][r % HT][lane];
            dx = dx + yp[1][v][r % HT][lane];
            e = e + yp[2][v][r % HT][lane];
          }
          const int t = tn + r;
          const bool there = t < stop;
          Row<T>(dzp + (int64_t)t * a.sdz.t, there && gate, k.cnt).put(gz[i] * fma(Dc, ur[i], y));
          const T dy = sy[r][lane], dd = fma(dx, ur[i], e * T(kLn2)) * ds[i];
          dD = fma(dy, ur[i], dD);
          dbias = dbias + dd;
          Row<T>(dup + (int64_t)t * a.sdu.t, there, k.cnt).put(fma(dx, sd[r][lane], Dc * dy));
          Row<T>(ddp + (int64_t)t * a.sddt.t, there, k.cnt).put(dd);
        }
        if (s > 0) __syncthreads();
      }
      const int rows = stop - t0 < TT ? stop - t0 : TT, gn = (int)(a.G * N) * (int)sizeof(T);
      const int64_t at = (prow + (int64_t)t0 * a.G) * N;
      const Rsrc rb = make_rsrc((const T*)a.dBp + at, rows * gn), rc = make_rsrc((const T*)a.dCp + at, rows * gn);
#pragma unroll
      for (int i = 0; i < In::MAPS; ++i) {
        const int f = threadIdx.x + 64 * W * i, r = f / NP, n = f % NP;
        const int off = n < N && r < TT ? r * gn + n * (int)sizeof(T) : -1;
        const int rr = TT * NP % (64 * W) != 0 && r >= TT ? 0 : r;
        store_at(rb, off, sg[rr][n]);
        store_at(rc, off, sg[rr][NP + n]);
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
  for (int64_t p = 0; p < parts; p += 8) {  // eight terms' loads in flight
    T x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = prm[(p + u < parts ? p + u : parts - 1) * (N + 2) * C + id];
#pragma unroll
    for (int u = 0; u < 8; ++u) s = p + u < parts ? s + x[u] : s;
  }
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
  for (int p = 0; p < a.tpg; p += 8) {  // sixteen loads in flight
    T vx[8], vy[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t at = (p + u < a.tpg ? p + u : a.tpg - 1) * n1 + id;
      vx[u] = ((const T*)a.dBp)[at];
      vy[u] = ((const T*)a.dCp)[at];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      x = p + u < a.tpg ? x + vx[u] : x;
      y = p + u < a.tpg ? y + vy[u] : y;
    }
  }
  dB[b * sB.b + t * sB.t + g * gB + n] = x;
  dC[b * sC.b + t * sC.t + g * gC + n] = y;
}

// One position per sequence, the states in place. A group of LPC lanes owns a
// channel, four states each; bound by reading and writing the states once (64 x
// 1536 x 16 float32, 14 MB: 5.6 us, launch included; the copy rate alone 2.7; float64 9).
template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(256) scan_step_kernel(ScanArgs a) {
  constexpr int NS = kStates;
  typedef T vt __attribute__((ext_vector_type(4)));
  const uint32_t bc = blockIdx.x * (256 / LPC) + threadIdx.x / LPC, b32 = bc / (uint32_t)a.C;
  const int64_t c = bc - b32 * (uint32_t)a.C, b = b32;
  const int n0 = (int)(threadIdx.x % LPC) * NS, N = (int)a.N;
  const bool on = b < a.B;
  T y = T(0);
  T u = T(0);
  if (on) {
    u = ((const T*)a.u)[b * a.su.b + c];
    T raw = ((const T*)a.dt)[b * a.sdt.b + c];
    if (a.bias) raw = raw + ((const T*)a.bias)[c];
    const T d = step_size(raw, a.softplus, true), x = d * u;
    const int64_t g = (uint32_t)c / (uint32_t)a.tpg;
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
          h[j] = fma(exp2_of(d * decay_rate(T(A[j]))), h[j], x * Bp[j]);
          y = fma(Cp[j], h[j], y);
        }
        *(vt*)hp = h;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (n0 + j < N) {
          const T h = fma(exp2_of(d * decay_rate(Ap[j])), hp[j], x * Bp[j]);
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

// Segments of T: one where the blocks (B * C / 64, of W waves) occupy the card. A
// split costs the exponentials a second time, so it pays while the card would run
// fewer than about four waves per CU (float64 three, whose exponentials cost
// more), but not beyond half a block per CU (sixteen waves fill one; the segments
// have to run at once) or two. Forward and backward of 1024 positions x 1536
// channels, us in one piece and cut, float32: 4 states, 384 blocks 917 / 504, 672
// blocks 921 / 892, 960 blocks 937 / 1222; 8 states, 288 blocks 785 / 459, 504
// blocks 800 / 751, 768 blocks 812 / 1106; 16 states, 192 blocks 503 / 376, 240
// blocks 506 / 495, 264 blocks 650 / 686; 32 states, 120 blocks 607 / 421, 192 blocks
// 612 / 789; 64 states, 120 blocks 1179 / 820, 192 blocks 1203 / 1568. float64: 8
// states, 384 blocks 1826 / 1798, 432 blocks 1830 / 2188; 16 states, 144 blocks 1296
// / 1093, 192 blocks 1302 / 1348; 64 states, 120 blocks 6957 / 4858. Then enough
// segments for 12 waves per CU (three blocks at 16 states), of at least two tiles each.
template <typename T>
static void scan_segments(ScanArgs& a, int TT, int W) {
  const int64_t cus = num_cus(), blocks = a.B * a.ct, want = (W <= 4 ? 12 / W : 2) * cus, tiles = cdiv(a.T, TT);
  const int64_t waves = (sizeof(T) == 4 ? 4 : 3) * cus / W;
  const int64_t full = waves < cus / 2 ? cus / 2 : waves > 2 * cus ? 2 * cus : waves;
  int64_t s = blocks >= full ? 1 : want / blocks;
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
  DTMI_CHECK(G * N < (1 << 23), "%s: %lld groups of %lld states", what, (long long)G, (long long)N);
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
  scan_segments<T>(a, tile_len<T>(W, false), W);
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

// The gradients of the maps from their channel tiles' terms (a.tpg tiles; none: zeros).
template <typename T>
static int scan_maps(const ScanArgs& a, void* dB, BT sdB, int64_t gdB, void* dC, BT sdC, int64_t gdC) {
  scan_map_kernel<T><<<(unsigned)cdiv(a.B * a.T * a.G * a.N, 256), 256, 0, stream()>>>(a, (T*)dB, sdB, gdB, (T*)dC, sdC,
                                                                                      gdC);
  LAUNCH_CHECK("scan: map gradients");
  return DTMI_OK;
}

template <typename T>
static int scan_bwd(ScanArgs& a, void* dA, void* dB, BT sdB, int64_t gdB, void* dC, BT sdC, int64_t gdC, void* dD,
                    void* dbias) {
  const int W = waves_for(a.N);
  scan_segments<T>(a, tile_len<T>(W, true), W);
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
    const hipError_t e = hipGetLastError();
    rc = e == hipSuccess ? scan_maps<T>(a, dB, sdB, gdB, dC, sdC, gdC) : fail_hip(e, "dtmi_scan_bwd", __FILE__, __LINE__);
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
  *count = B * cdiv(T, kKeep) * N * C;
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
  const size_t es = dtype == DTMI_F32 ? 4 : 8;
  if (C == 0) {  // the maps alone have gradients, of no terms
    if (B == 0 || T == 0) return DTMI_OK;
    DTMI_CHECK(dB && dC && dB_strides && dC_strides, "dtmi_scan_bwd: NULL operand");
    DTMI_CHECK(B * T * G * N <= (int64_t)0x7fffffff * 256, "dtmi_scan_bwd: too many elements");
    ScanArgs a{};
    a.B = B, a.T = T, a.N = N, a.G = G;
    const BT sdB = bt(dB_strides), sdC = bt(dC_strides);
    return dtype == DTMI_F32 ? scan_maps<float>(a, dB, sdB, dB_strides[2], dC, sdC, dC_strides[2])
                             : scan_maps<double>(a, dB, sdB, dB_strides[2], dC, sdC, dC_strides[2]);
  }
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
  DTMI_CHECK(B * C < ((int64_t)1 << 31), "dtmi_scan_step: too many elements");
  ScanArgs a{};
  a.u = u, a.dt = dt, a.A = A, a.Bm = Bm, a.Cm = Cm, a.D = D, a.z = z, a.bias = dt_bias, a.hT = state, a.out = out;
  a.su.b = u_stride, a.sdt.b = dt_stride, a.sz.b = z_stride, a.sout.b = out_stride;
  a.sB.b = B_strides[0], a.gB = B_strides[1], a.sC.b = C_strides[0], a.gC = C_strides[1];
  a.B = B, a.C = C, a.N = N, a.G = G, a.softplus = softplus, a.tpg = (int)(C / G);
  TimedLaunch tl(DTMI_FAM_OTHER, 7.0 * B * C * N);
  if (dtype == DTMI_F32)
    scan_step<float>(a);
  else
    scan_step<double>(a);
  LAUNCH_CHECK("dtmi_scan_step");
  return DTMI_OK;
  DTMI_BODY_END
}
