// Attention to another sequence's states: o = softmax(q k^T scale) v over the
// first lengths[b] of Tk keys, with H query heads sharing Hk key/value heads
// (head h reads h / (H / Hk)). A row whose memory is empty is 0 and passes
// no gradient; keys past the length are never read.
//
// The queries of all heads that share a key/value head form one matrix of
// R = (H / Hk) Tq rows (row r: head r / Tq of the group, query r % Tq), so one
// query token with shared heads fills the columns of a matrix tile, and dK and
// dV sum over the heads that share them in the loop over rows, without atomics.
//
// Tiles of 16 x 16 x 4 MFMAs in the transposed formulation of the causal
// kernels: the operand a wave owns (queries in the forward and the dQ pass,
// keys in the dK/dV pass) is the tile's columns and stays in registers; the
// other operand passes through LDS, shared by the block's four waves. A
// result register i of lane group g then is what that lane feeds to the next
// product as its slot g of step i, with the other operand read from LDS at row
// row(i, g).
//
// Forward: scores in base 2, a reference maximum per query that moves only
// when a score exceeds it by 2^8, sum and output rescaled then. A score is scaled
// and rounded as the reference was before it is subtracted: in one rounding with
// the difference, scores of 2^32 and more would leave the reference's own
// rounding, hundreds, in the exponent. Backward: the
// probabilities from the forward's reference and sum (the same products in the
// same order, so the same scores), dV += P^T dO, dP = dO V^T, dS = P (dP -
// rowsum(dO O)), dK += dS^T Q in the pass over keys; S, dP and dQ = dS K in
// the pass over queries. A memory of one key has P = 1 whatever the score, so dS,
// dQ and dK are 0: dP and rowsum(dO O), the same sum in two orders, would leave
// their rounding.
//
// Few rows or few keys give few blocks: the loop (over keys in the forward and
// the dQ pass, over rows in the dK/dV pass) is then split over blocks, whose
// partial results a small kernel joins in a fixed order.
#include <cmath>

#include "bufrsrc.h"
#include "common.h"

namespace dtmi {

template <typename T>
struct XM;
template <>
struct XM<float> {
  static constexpr int VEC = 4, PAD = 4;
  typedef float acc_t __attribute__((ext_vector_type(4)));
  typedef float vec_t __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ acc_t mma(float a, float b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int i, int g) { return 4 * g + i; }
  static __device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
  static constexpr float lowest = -3.40282347e38f;
};
template <>
struct XM<double> {
  static constexpr int VEC = 2, PAD = 2;
  typedef double acc_t __attribute__((ext_vector_type(4)));
  typedef double vec_t __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ acc_t mma(double a, double b, acc_t c) {
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int i, int g) { return g + 4 * i; }
  static __device__ __forceinline__ double ex2(double x) { return exp2(x); }
  static constexpr double lowest = -1.7976931348623157e308;
};

struct HT {
  int64_t b, h, t;
};

// Division by a fixed d >= 1 of numbers below 2^31 as a multiplication
// (Granlund and Montgomery, 1994): n / d = (mulhi(n, m) + n) >> l.
struct FastDiv {
  uint32_t m, l, d;
  FastDiv() = default;
  explicit FastDiv(uint32_t d_) : d(d_) {
    l = 0;
    while ((1ull << l) < d) ++l;
    m = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> l; }
};

struct XArgs {
  const void *q, *k, *v, *o, *dO;
  void *out, *dq, *dk, *dv;
  void *rowmax, *rowsum;  // [B, H, Tq]: the reference maximum (base 2) and the sum against it
  void* drow;             // [B, H, Tq]: rowsum(dO O)
  void *po, *pm, *pl;     // partial results of a split loop
  void* ds;               // dS for the dQ pass, or NULL: 16 x 16 tiles [B, Hk][rows / 16][keys / 16], each [key][4 g + i] for row(i, g)
  int64_t rt, kt;         // its tiles of rows and keys
  const int64_t* lengths;
  HT sq, sk, sv, so, sdo, sdq, sdk, sdv;
  int64_t B, H, Hk, G, Tq, Tk, D, R;  // G: heads per group, H / Hk; R: rows, G Tq
  double scale;
  FastDiv by_tq;  // rows to heads
  int nsplit;   // parts of the loop, at most
  int per, step;  // positions per part, a multiple of step
  int parts;      // with lengths: parts of all sequences together
  int ntile;    // blocks along the owned axis
  int vec;      // 16-byte loads and stores allowed for every operand, positions less than 2^23 elements apart
};

__device__ __forceinline__ int64_t key_count(const XArgs& a, int64_t b) {
  if (!a.lengths) return a.Tk;
  const int64_t n = a.lengths[b];
  return n < 0 ? 0 : n > a.Tk ? a.Tk : n;
}

// First element of a group's rows in an array with strides s, and row r's offset from there
template <typename T>
__device__ __forceinline__ T* group_of(const XArgs& a, const void* p, const HT& s, int64_t b, int64_t kh) {
  return (T*)p + b * s.b + kh * a.G * s.h;
}
__device__ __forceinline__ int64_t row_at(const XArgs& a, const HT& s, int r) {
  const uint32_t h = a.by_tq.div((uint32_t)r), t = (uint32_t)r - h * a.by_tq.d;
  return (int64_t)h * s.h + (int64_t)t * s.t;
}
__device__ __forceinline__ int64_t stat_at(const XArgs& a, int64_t b, int64_t kh, int r) {
  return (b * a.H + kh * a.G) * a.Tq + r;
}

// The d that tile column m of 16 stands for in the N products along D: chunks of
// products as wide as a vector allows (5: 4 + 1), each 16 vectors of the row in
// order, so that the lanes' reads are contiguous (6 as 4 + 2: forward and backward
// of 8 x 12 heads x 1024 x 512 x 96 672 us, as 6 elements a lane 738).
template <typename T, int N>
struct Cols {
  static constexpr int V = XM<T>::VEC, FULL = N / V * V, TWO = FULL + ((N - FULL) & 2);
  static __device__ constexpr int width(int t) { return t < FULL ? V : t < TWO ? 2 : 1; }
  static __device__ constexpr int first(int t) { return t < FULL ? t / V * V : t < TWO ? FULL : TWO; }  // product of t's chunk
  static __device__ __forceinline__ int d(int t, int m) { return 16 * first(t) + width(t) * m + (t - first(t)); }
};

// A lane's slice of one row as MFMA operand: element e of vector f is
// d = 4 VEC f + VEC g + e, so the lane groups' reads of a row are contiguous.
template <typename T, int DP>
__device__ __forceinline__ void load_slice(typename XM<T>::vec_t (&f)[DP / (4 * XM<T>::VEC)], const T* __restrict__ row,
                                           bool in, int D, int g, bool vec) {
  constexpr int VEC = XM<T>::VEC;
  typedef typename XM<T>::vec_t VT;
#pragma unroll
  for (int i = 0; i < DP / (4 * VEC); ++i) {
    const int d = 4 * VEC * i + VEC * g;
    VT x = VT(0);
    if (vec) {
      if (in && d < D) x = *reinterpret_cast<const VT*>(row + d);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (in && d + e < D) x[e] = row[d + e];
    }
    f[i] = x;
  }
}

// NR rows of a tile on their way from global memory to LDS [NR][DP + PAD];
// rows that do not exist and columns at and past D are zero.
// VEC: 16-byte loads, and rows that 32 bits reach from a tile's first.
template <typename T, int NR, int DP, bool VEC>
struct Rows {
  typedef typename XM<T>::vec_t VT;
  static constexpr int V = XM<T>::VEC, LD = DP + XM<T>::PAD, ALL = NR * DP / V, NV = (ALL + 255) / 256;
  VT x[NV];
  uint32_t off[NV];  // bytes from the tile's first row; past every buffer's end in columns from D on
  static __device__ __forceinline__ int row(int i) { return (threadIdx.x + 256 * i) / (DP / V); }
  static __device__ __forceinline__ int col(int i) { return (threadIdx.x + 256 * i) % (DP / V) * V; }
  static __device__ __forceinline__ bool mine(int i) { return ALL % 256 == 0 || threadIdx.x + 256 * i < ALL; }
  __device__ __forceinline__ void start(int64_t st, int D) {
#pragma unroll
    for (int i = 0; i < NV; ++i) off[i] = mine(i) && col(i) < D ? (uint32_t)((row(i) * st + col(i)) * sizeof(T)) : 0x80000000u;
  }
  // `n` rows from p on, `st` elements apart (start()): the buffer ends with the
  // last of them, so the address work of a tile is scalar
  __device__ __forceinline__ void fetch(const T* p, int64_t st, int n, int D) {
    if constexpr (VEC) {
      n = n < NR ? n : NR;
      const Rsrc r = make_rsrc(p, n > 0 ? (uint64_t)(((n - 1) * st + D) * sizeof(T)) : 0);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        x[i] = __builtin_bit_cast(VT, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off[i], 0, 0));
    } else {
      gather([&](int i) { return i < n ? p + i * st : nullptr; }, D);
    }
  }
  // rows at base(r), NULL for none
  template <typename F>
  __device__ __forceinline__ void gather(const F& base, int D) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const T* p = mine(i) ? base(row(i)) : nullptr;
      const int d = col(i);
      VT v = VT(0);
      if (VEC) {
        if (p && d < D) v = *reinterpret_cast<const VT*>(p + d);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (p && d + e < D) v[e] = p[d + e];
      }
      x[i] = v;
    }
  }
  __device__ __forceinline__ void put(T* __restrict__ lds) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (mine(i)) *reinterpret_cast<VT*>(lds + row(i) * LD + col(i)) = x[i];
  }
};

// A row's elements Cols::d(t, c), as vectors; f (of a vector's first d): whether it is there
template <typename T, int N, typename F>
__device__ __forceinline__ void row_cols(T (&x)[N], const T* __restrict__ row, int c, const F& f) {
  using L = Cols<T, N>;
#pragma unroll
  for (int t = 0; t < N; ++t) {
    if (t != L::first(t)) continue;
    const int d = L::d(t, c);
    if (L::width(t) == XM<T>::VEC) {
      typename XM<T>::vec_t y = typename XM<T>::vec_t(0);
      if (f(d)) y = *reinterpret_cast<const typename XM<T>::vec_t*>(row + d);
#pragma unroll
      for (int e = 0; e < XM<T>::VEC; ++e) x[t + e] = y[e];
    } else if (L::width(t) == 2) {
      typedef T v2 __attribute__((ext_vector_type(2)));
      v2 y = v2(0);
      if (f(d)) y = *reinterpret_cast<const v2*>(row + d);
      x[t] = y[0];
      if (t + 1 < N) x[t + 1] = y[1];
    } else {
      x[t] = f(d) ? row[d] : T(0);
    }
  }
}
// A lane's slice of row r0 + c of an LDS tile, and its columns Cols::d(t, c) of
// the rows row(i, g): the two ways a tile's rows enter a product.
template <typename T, int DP>
__device__ __forceinline__ void lds_slice(typename XM<T>::vec_t (&x)[DP / (4 * XM<T>::VEC)], const T* __restrict__ lds, int r0,
                                          int g, int c) {
  constexpr int VEC = XM<T>::VEC, LD = DP + XM<T>::PAD;
#pragma unroll
  for (int i = 0; i < DP / (4 * VEC); ++i)
    x[i] = *reinterpret_cast<const typename XM<T>::vec_t*>(lds + (r0 + c) * LD + 4 * VEC * i + VEC * g);
}
template <typename T, int DP>
__device__ __forceinline__ void lds_cols(T (&x)[4][DP / 16], const T* __restrict__ lds, int r0, int g, int c) {
  constexpr int N = DP / 16, LD = DP + XM<T>::PAD;
#pragma unroll
  for (int i = 0; i < 4; ++i) row_cols<T, N>(x[i], lds + (r0 + XM<T>::row(i, g)) * LD, c, [](int) { return true; });
}
// Two 16 x 16 tiles of products of slices, their chains of dependent MFMAs interleaved
template <typename T, int NF>
__device__ __forceinline__ void mul_slices(typename XM<T>::acc_t& p, const typename XM<T>::vec_t (&xp)[NF],
                                           const typename XM<T>::vec_t (&fp)[NF], typename XM<T>::acc_t& q,
                                           const typename XM<T>::vec_t (&xq)[NF], const typename XM<T>::vec_t (&fq)[NF]) {
  p = q = typename XM<T>::acc_t(0);
#pragma unroll
  for (int i = 0; i < NF; ++i)
#pragma unroll
    for (int e = 0; e < XM<T>::VEC; ++e) {
      p = XM<T>::mma(xp[i][e], fp[i][e], p);
      q = XM<T>::mma(xq[i][e], fq[i][e], q);
    }
}
// out^T (d by column) += sum over a tile's 16 rows of x(row, d) p(row, column)
template <typename T, int N>
__device__ __forceinline__ void mul_cols(typename XM<T>::acc_t (&out)[N], const T (&x)[4][N],
                                         const typename XM<T>::acc_t& p) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < N; ++t) out[t] = XM<T>::mma(x[i][t], p[i], out[t]);
}
// float64 products' operands are read when the ones before are done with: read
// ahead, as the compiler prefers, they spill. float32 has the registers.
template <typename T>
__device__ __forceinline__ void phase() {
  if constexpr (sizeof(T) == 8) __builtin_amdgcn_sched_barrier(0);
}

// The lane's part of a result row: registers (t, i) are Cols::d(t, row(i, g))
template <typename T, int DP>
__device__ __forceinline__ void put_row(T* __restrict__ row, const typename XM<T>::acc_t (&x)[DP / 16], T mul, int D,
                                        int g, bool vec) {
  constexpr int N = DP / 16;
  using L = Cols<T, N>;
  typedef typename XM<T>::vec_t VT;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < N; ++t) {
      const int d = L::d(t, XM<T>::row(i, g));
      if (vec && L::width(t) == XM<T>::VEC) {
        if (t % XM<T>::VEC != 0) continue;
        VT y;
#pragma unroll
        for (int e = 0; e < XM<T>::VEC; ++e) y[e] = x[t + e][i] * mul;
        if (d < D) *reinterpret_cast<VT*>(row + d) = y;
      } else if (d < D) {
        row[d] = x[t][i] * mul;
      }
    }
}

// The result and the gradient of a row without a finite score (weight 0) are 0,
// whatever infinite keys or values made of its products
template <typename T, int N>
__device__ __forceinline__ void none_without(typename XM<T>::acc_t (&x)[N], T weight) {
  if (weight == T(0))
#pragma unroll
    for (int t = 0; t < N; ++t) x[t] = typename XM<T>::acc_t(0);
}

template <typename T>
__device__ __forceinline__ T over_groups_max(T x) {
  x = fmax(x, __shfl_xor(x, 16, 64));
  return fmax(x, __shfl_xor(x, 32, 64));
}
template <typename T>
__device__ __forceinline__ T over_groups_sum(T x) {
  x = x + __shfl_xor(x, 16, 64);
  return x + __shfl_xor(x, 32, 64);
}

struct XBlock {
  int64_t b, kh;
  int tile, split;
  // this block's part of a loop over n positions, `per` to a part
  __device__ __forceinline__ bool part(int per, int n, int& lo, int& hi) const {
    const int64_t from = (int64_t)split * per;
    lo = from < n ? (int)from : n;
    hi = n - lo > per ? lo + per : n;
    return lo < hi || split == 0;
  }
};
// Keys per part of a loop over keys: the host's, or with lengths such that all
// sequences' parts together number a.parts per key/value head, so that a long
// sequence gets more blocks and not longer ones (every wave sums the lengths).
// In 32 bits (the host checks that the lengths' sum fits) and known to be one value:
// as lanes' 64-bit numbers they kept the loop's bounds in vector registers and cost
// the forward of 4 x 8 / 2 heads x 333 x 1501 x 72, padded, 4 us of 57.
__device__ __forceinline__ int keys_per_part(const XArgs& a) {
  if (!a.lengths || a.nsplit == 1) return a.per;
  uint32_t total = 0;
  for (int b = threadIdx.x & 63; b < (int)a.B; b += 64) total += (uint32_t)key_count(a, b);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) total += __shfl_xor(total, x, 64);
  total = (uint32_t)__builtin_amdgcn_readfirstlane((int)total);
  const uint32_t parts = (uint32_t)a.parts, split = (uint32_t)a.nsplit, step = (uint32_t)a.step;
  const uint32_t fair = (total + parts - 1) / parts, least = ((uint32_t)a.Tk + split - 1) / split;
  return (int)(((fair > least ? fair : least) + step - 1) / step * step);
}
__device__ __forceinline__ XBlock x_block(const XArgs& a) {
  // blocks are dealt to the eight XCDs in turn: XCD x takes the x-th eighth of
  // the blocks, so that those sharing a head's keys share an L2 (forward of 8 x 12
  // heads x 1024 x 2048 x 64: 457 us, in the dealt order 463); not with lengths,
  // where an eighth may hold the long sequences (4 x 8 / 2 heads x 333 x 777 x 72,
  // forward and backward: 427 us so and 314 dealt, when this was chosen)
  const unsigned n = gridDim.x, xcd = blockIdx.x & 7, more = n & 7;
  const unsigned id = a.lengths ? blockIdx.x : xcd * (n >> 3) + (xcd < more ? xcd : more) + (blockIdx.x >> 3);
  XBlock k;
  const unsigned r = id / (unsigned)a.ntile, bh = r / (unsigned)a.nsplit;
  k.tile = (int)(id - r * (unsigned)a.ntile);
  k.split = (int)(r - bh * (unsigned)a.nsplit);
  k.b = bh / (unsigned)a.Hk;
  k.kh = bh % (unsigned)a.Hk;
  return k;
}

// Waves per SIMD the registers are cut to: more than two would spill, and the
// wide float64 tiles do at two, those of the pass that owns two operands (kv) from
// 64 elements on (backward of 8 x 12 heads x 1024 x 512 x 64: 937 us at two, 735).
// (With no bound the accumulators go to the accumulation registers and every use
// of a score is a move more: forward and backward of the same in float32 took 671
// us so, and 582 bounded.)
template <typename T>
constexpr int x_waves(int DP, bool kv = false) {
  return sizeof(T) == 8 && DP >= (kv ? 64 : 80) ? 1 : 2;
}

constexpr int kKeys = 32;  // keys (rows, in the dK/dV pass) per tile

// The forward for more than 16 rows: a wave owns 16 of them. Bound by the MFMAs:
// two products, 4 D per score. float32, 32 x 12 heads x 1024 x 2048 x 64: 128
// TFLOP/s (a large library product: 154); 8 x 12 x 1024 x 512: 115 us, 112: of 1536
// blocks four waves per SIMD (103 registers) take 1024 at once, and the second round is
// half empty. float64 263 us, 49 (a large product 73). Five or six waves per SIMD
// spill; a second LDS buffer and 32 rows per wave gave nothing.
template <typename T, int DP, bool VEC>
__global__ void __launch_bounds__(256, x_waves<T>(DP)) xattn_fwd_kernel(XArgs a) {
  using M = XM<T>;
  typedef typename M::acc_t AT;
  constexpr int N = DP / 16, LD = DP + M::PAD, KT = kKeys;
  __shared__ __attribute__((aligned(16))) T Ks[KT * LD], Vs[KT * LD];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15, D = (int)a.D;
  const XBlock k = x_block(a);
  const int len = (int)key_count(a, k.b);
  int lo, hi;
  if (!k.part(keys_per_part(a), len, lo, hi)) return;
  const int r0 = (k.tile * 4 + w) * 16, R = (int)a.R, r = r0 + c;
  const T* Qb = group_of<const T>(a, a.q, a.sq, k.b, k.kh);
  typename M::vec_t qf[DP / (4 * M::VEC)];
  load_slice<T, DP>(qf, Qb + (r < R ? row_at(a, a.sq, r) : 0), r < R, D, g, VEC);
  const T* Kb = (const T*)a.k + k.b * a.sk.b + k.kh * a.sk.h;
  const T* Vb = (const T*)a.v + k.b * a.sv.b + k.kh * a.sv.h;
  Rows<T, KT, DP, VEC> fk, fv;
  if constexpr (VEC) {
    fk.start(a.sk.t, D);
    fv.start(a.sv.t, D);
  }
  auto fetch = [&](int j0) {
    fk.fetch(Kb + j0 * a.sk.t, a.sk.t, hi - j0, D);
    fv.fetch(Vb + j0 * a.sv.t, a.sv.t, hi - j0, D);
  };
  const T sl2 = (T)(a.scale * 1.4426950408889634);
  AT o[N];
  T mref = M::lowest, l = T(0);
#pragma unroll
  for (int t = 0; t < N; ++t) o[t] = AT(0);
  const bool busy = r0 < R;
  if (lo < hi) {
    fetch(lo);
    fk.put(Ks);
    fv.put(Vs);
  }
  __syncthreads();
  for (int j0 = lo; j0 < hi; j0 += KT) {
    const bool more = j0 + KT < hi;
    if (more) fetch(j0 + KT);
    if (busy) {
      constexpr int NF = DP / (4 * M::VEC);
      typename M::vec_t x0[NF], x1[NF];
      T v0[4][N], v1[4][N];
      AT p0, p1;
      lds_slice<T, DP>(x0, Ks, 0, g, c);
      lds_slice<T, DP>(x1, Ks, 16, g, c);
      mul_slices<T, NF>(p0, x0, qf, p1, x1, qf);
      phase<T>();
      lds_cols<T, DP>(v0, Vs, 0, g, c);
      T top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in0 = more || j0 + M::row(i, g) < hi, in1 = more || j0 + 16 + M::row(i, g) < hi;
        p0[i] = in0 ? p0[i] * sl2 : -INFINITY;
        p1[i] = in1 ? p1[i] * sl2 : -INFINITY;
        top = fmax(top, fmax(p0[i], p1[i]));
      }
      if (__any(top > mref + T(8))) {
        const T next = fmax(mref, over_groups_max(top));
        const T alpha = M::ex2(mref - next);
        l = l * alpha;
#pragma unroll
        for (int t = 0; t < N; ++t) o[t] *= alpha;
        mref = next;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p0[i] = M::ex2(p0[i] - mref);
        p1[i] = M::ex2(p1[i] - mref);
        l = l + (p0[i] + p1[i]);
      }
      mul_cols<T, N>(o, v0, p0);
      phase<T>();
      lds_cols<T, DP>(v1, Vs, 16, g, c);
      mul_cols<T, N>(o, v1, p1);
    }
    __syncthreads();
    if (more) {
      fk.put(Ks);
      fv.put(Vs);
    }
    __syncthreads();
  }
  const T sum = over_groups_sum(l);
  if (r >= R) return;
  if (a.nsplit > 1) {
    const int64_t at = ((k.b * a.Hk + k.kh) * a.nsplit + k.split) * a.R + r;
    put_row<T, DP>((T*)a.po + at * DP, o, T(1), DP, g, true);
    if (g == 0) {
      ((T*)a.pm)[at] = mref;
      ((T*)a.pl)[at] = sum;
    }
    return;
  }
  none_without<T, N>(o, sum);
  put_row<T, DP>(group_of<T>(a, a.out, a.so, k.b, k.kh) + row_at(a, a.so, r), o, sum == T(0) ? T(0) : T(1) / sum, D, g, VEC);
  if (g == 0 && a.rowmax) {
    const int64_t at = stat_at(a, k.b, k.kh, r);
    ((T*)a.rowmax)[at] = mref;
    ((T*)a.rowsum)[at] = sum;
  }
}

// Up to 16 rows per key/value head (one query token with shared heads): bound
// by reading k and v once. Each wave takes every fourth 16 keys of the block's
// part and loads them straight into the products' operand registers, the next
// 16 while it works; the waves' results are joined through LDS. One query of
// 64 x 12 heads x 1024 keys x 64, 403 MB: 74 us, 5.4 TB/s (the kernel for more
// rows, three of its waves idle: 84); of 8 x 16 / 4 heads x 4999 x 128: 34 and 56. In
// float64 148 and 82.
template <typename T, int DP, bool VEC>
__global__ void __launch_bounds__(256, x_waves<T>(DP)) xattn_rows_kernel(XArgs a) {
  using M = XM<T>;
  typedef typename M::acc_t AT;
  typedef typename M::vec_t VT;
  constexpr int N = DP / 16, NF = DP / (4 * M::VEC);
  __shared__ T so[4][16][DP + 1], sm[4][16], sl[4][16];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15, D = (int)a.D, R = (int)a.R;
  const XBlock k = x_block(a);
  const int len = (int)key_count(a, k.b);
  int lo, hi;
  if (!k.part(keys_per_part(a), len, lo, hi)) return;
  const T* Qb = group_of<const T>(a, a.q, a.sq, k.b, k.kh);
  VT qf[NF];
  load_slice<T, DP>(qf, Qb + (c < R ? row_at(a, a.sq, c) : 0), c < R, D, g, VEC);
  const T* Kb = (const T*)a.k + k.b * a.sk.b + k.kh * a.sk.h;
  const T* Vb = (const T*)a.v + k.b * a.sv.b + k.kh * a.sv.h;
  auto fetch = [&](VT(&x)[NF], T(&v)[4][N], int j) {
    load_slice<T, DP>(x, Kb + (int64_t)(j + c < hi ? j + c : 0) * a.sk.t, j + c < hi, D, g, VEC);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = j + M::row(i, g);
      const T* row = Vb + (int64_t)(r < hi ? r : 0) * a.sv.t;
      if (VEC) {
        row_cols<T, N>(v[i], row, c, [&](int d) { return r < hi && d < D; });
      } else {
#pragma unroll
        for (int t = 0; t < N; ++t) {
          const int d = Cols<T, N>::d(t, c);
          v[i][t] = r < hi && d < D ? row[d] : T(0);
        }
      }
    }
  };
  const T sl2 = (T)(a.scale * 1.4426950408889634);
  AT o[N];
  T mref = M::lowest, l = T(0);
#pragma unroll
  for (int t = 0; t < N; ++t) o[t] = AT(0);
  VT x[NF], nx[NF];
  T v[4][N], nv[4][N];
  if (lo + 16 * w < hi) fetch(x, v, lo + 16 * w);
  for (int j = lo + 16 * w; j < hi; j += 64) {
    if (j + 64 < hi) fetch(nx, nv, j + 64);
    AT s = AT(0);
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
      for (int e = 0; e < M::VEC; ++e) s = M::mma(x[i][e], qf[i][e], s);
    T top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = j + M::row(i, g) < hi ? s[i] * sl2 : -INFINITY;
      top = fmax(top, s[i]);
    }
    if (__any(top > mref + T(8))) {
      const T next = fmax(mref, over_groups_max(top));
      const T alpha = M::ex2(mref - next);
      l = l * alpha;
#pragma unroll
      for (int t = 0; t < N; ++t) o[t] *= alpha;
      mref = next;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = M::ex2(s[i] - mref);
      l = l + s[i];
    }
    mul_cols<T, N>(o, v, s);
#pragma unroll
    for (int i = 0; i < NF; ++i) x[i] = nx[i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < N; ++t) v[i][t] = nv[i][t];
  }
  const T sum = over_groups_sum(l);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < N; ++t) so[w][c][Cols<T, N>::d(t, M::row(i, g))] = o[t][i];
  if (g == 0) {
    sm[w][c] = mref;
    sl[w][c] = sum;
  }
  __syncthreads();
  for (int f = threadIdx.x; f < R * DP; f += 256) {
    const int r = f / DP, d = f % DP;
    T top = sm[0][r];
#pragma unroll
    for (int u = 1; u < 4; ++u) top = fmax(top, sm[u][r]);
    T y = T(0), tot = T(0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const T wt = sm[u][r] == top ? T(1) : M::ex2(sm[u][r] - top);
      y = fma(so[u][r][d], wt, y);
      tot = fma(sl[u][r], wt, tot);
    }
    if (a.nsplit > 1) {
      const int64_t at = ((k.b * a.Hk + k.kh) * a.nsplit + k.split) * a.R + r;
      ((T*)a.po)[at * DP + d] = y;
      if (d == 0) {
        ((T*)a.pm)[at] = top;
        ((T*)a.pl)[at] = tot;
      }
    } else {
      if (d < D) (group_of<T>(a, a.out, a.so, k.b, k.kh) + row_at(a, a.so, r))[d] = tot == T(0) ? T(0) : y / tot;
      if (d == 0 && a.rowmax) {
        ((T*)a.rowmax)[stat_at(a, k.b, k.kh, r)] = top;
        ((T*)a.rowsum)[stat_at(a, k.b, k.kh, r)] = tot;
      }
    }
  }
}

// Parts of a sequence's keys (0 keys: one, of zeros).
__device__ __forceinline__ int part_count(const XArgs& a, int64_t b) {
  const int per = keys_per_part(a), len = (int)key_count(a, b);
  return len > per ? (len + per - 1) / per : 1;
}

// Joins the forward's parts (at most 64) of few rows: a block per row. Lane s
// weighs part s; then 256 / DP groups of threads over d add every so many parts
// each, eight loads in flight, and their sums are added in order. (32 parts of
// 128 rows: 4.0 us, a wave per row 7.8; of 10656 rows 17.5 and 9.9.)
template <typename T, int DP>
__global__ void __launch_bounds__(256) xattn_join_few_kernel(XArgs a) {
  constexpr int G = DP <= 32 ? 8 : DP <= 64 ? 4 : 2;
  __shared__ T swt[64], ssum, part[G][DP];
  const int64_t bh = blockIdx.x / (unsigned)a.R;
  const int r = (int)(blockIdx.x % (unsigned)a.R), lane = threadIdx.x & 63;
  const int64_t b = bh / a.Hk, kh = bh % a.Hk, at = bh * a.nsplit * a.R + r;
  const int n = part_count(a, b);
  if (threadIdx.x < 64) {
    const bool mine = lane < n;
    const T m = mine ? ((const T*)a.pm)[at + lane * a.R] : XM<T>::lowest;
    T top = m;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmax(top, __shfl_xor(top, x, 64));
    const T wt = m == top ? T(1) : XM<T>::ex2(m - top);
    T sum = mine ? ((const T*)a.pl)[at + lane * a.R] * wt : T(0);
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum = sum + __shfl_xor(sum, x, 64);
    swt[lane] = wt;
    if (lane == 0) {
      ssum = sum;
      if (a.rowmax) {
        ((T*)a.rowmax)[stat_at(a, b, kh, r)] = top;
        ((T*)a.rowsum)[stat_at(a, b, kh, r)] = sum;
      }
    }
  }
  const int d = threadIdx.x % DP, grp = threadIdx.x / DP;
  const T* p = (const T*)a.po + at * DP + d;
  T y = T(0), x[8];
  auto load = [&](int s) {
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = p[(int64_t)(s + G * u < n ? s + G * u : n - 1) * a.R * DP];
  };
  load(grp);  // ahead of the weights
  __syncthreads();
  if (grp < G) {
    for (int s = grp; s < n; s += 8 * G) {
      if (s != grp) load(s);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (s + G * u < n) y = fma(x[u], swt[s + G * u], y);
    }
    part[grp][d] = y;
  }
  __syncthreads();
  if (grp == 0 && d < a.D) {
    y = T(0);
#pragma unroll
    for (int u = 0; u < G; ++u) y = y + part[u][d];
    (group_of<T>(a, a.out, a.so, b, kh) + row_at(a, a.so, r))[d] = ssum == T(0) ? T(0) : y / ssum;
  }
}

// The same for many rows: a wave per row.
template <typename T, int DP>
__global__ void __launch_bounds__(256) xattn_join_kernel(XArgs a) {
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), bh = id / a.R;
  const int r = (int)(id % a.R);
  if (bh >= a.B * a.Hk) return;
  const int lane = threadIdx.x & 63;
  const int64_t b = bh / a.Hk, kh = bh % a.Hk, at = bh * a.nsplit * a.R + r;
  const int n = part_count(a, b);
  const bool mine = lane < n;
  const T m = mine ? ((const T*)a.pm)[at + lane * a.R] : XM<T>::lowest;
  T top = m;
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmax(top, __shfl_xor(top, x, 64));
  const T wt = m == top ? T(1) : XM<T>::ex2(m - top);
  T sum = mine ? ((const T*)a.pl)[at + lane * a.R] * wt : T(0);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) sum = sum + __shfl_xor(sum, x, 64);
  const T inv = sum == T(0) ? T(0) : T(1) / sum;
  T* out = group_of<T>(a, a.out, a.so, b, kh) + row_at(a, a.so, r);
#pragma unroll
  for (int e = 0; e < (DP + 63) / 64; ++e) {
    const int d = lane + 64 * e < DP ? lane + 64 * e : DP - 1;
    const T* p = (const T*)a.po + at * DP + d;
    T y = T(0);
    for (int s = 0; s < n; s += 8) {
      T x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = p[(int64_t)(s + u < n ? s + u : n - 1) * a.R * DP];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const T f = __shfl(wt, s + u < n ? s + u : 0, 64);
        if (s + u < n) y = fma(x[u], f, y);
      }
    }
    if (lane + 64 * e < a.D) out[lane + 64 * e] = sum == T(0) ? T(0) : y * inv;
  }
  if (lane == 0 && a.rowmax) {
    ((T*)a.rowmax)[stat_at(a, b, kh, r)] = top;
    ((T*)a.rowsum)[stat_at(a, b, kh, r)] = sum;
  }
}

// rowsum(dO O): 16 lanes per row; reads both once (8 x 12 x 1024 x 64 float32: 13 us, 3.8 TB/s)
template <typename T>
__global__ void __launch_bounds__(256) xattn_drow_kernel(XArgs a) {
  const int64_t id = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), bh = id / a.R;
  const int r = (int)(id % a.R);
  const bool on = bh < a.B * a.Hk;
  T s = T(0);
  if (on) {
    const int64_t b = bh / a.Hk, kh = bh % a.Hk;
    const T* o = group_of<const T>(a, a.o, a.so, b, kh) + row_at(a, a.so, r);
    const T* g = group_of<const T>(a, a.dO, a.sdo, b, kh) + row_at(a, a.sdo, r);
    for (int d = threadIdx.x & 15; d < a.D; d += 16) s = fma(o[d], g[d], s);
  }
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) s = s + __shfl_xor(s, m, 64);
  if (on && (threadIdx.x & 15) == 0) ((T*)a.drow)[stat_at(a, bh / a.Hk, bh % a.Hk, r)] = s;
}

// dQ where dS is not kept: a wave owns 16 rows and loops over the keys of its
// part. Bound by the MFMAs (three products): float32, 32 x 12 heads x 1024 x 2048 x
// 64, 131 TFLOP/s.
template <typename T, int DP, bool VEC>
__global__ void __launch_bounds__(256, x_waves<T>(DP)) xattn_bwd_q_kernel(XArgs a) {
  using M = XM<T>;
  typedef typename M::acc_t AT;
  constexpr int N = DP / 16, LD = DP + M::PAD, KT = kKeys, NF = DP / (4 * M::VEC);
  __shared__ __attribute__((aligned(16))) T Ks[KT * LD], Vs[KT * LD];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15, D = (int)a.D;
  const XBlock k = x_block(a);
  const int len = (int)key_count(a, k.b);
  int lo, hi;
  if (!k.part(keys_per_part(a), len, lo, hi)) return;
  if (len == 1) hi = lo;  // dS is 0
  const int r0 = (k.tile * 4 + w) * 16, R = (int)a.R, r = r0 + c;
  const bool in = r < R;
  const T* Qb = group_of<const T>(a, a.q, a.sq, k.b, k.kh);
  const T* Gb = group_of<const T>(a, a.dO, a.sdo, k.b, k.kh);
  typename M::vec_t qf[NF], gf[NF];
  load_slice<T, DP>(qf, Qb + (in ? row_at(a, a.sq, r) : 0), in, D, g, VEC);
  load_slice<T, DP>(gf, Gb + (in ? row_at(a, a.sdo, r) : 0), in, D, g, VEC);
  const int64_t st = stat_at(a, k.b, k.kh, in ? r : 0);
  const T sum = ((const T*)a.rowsum)[st], m = ((const T*)a.rowmax)[st], dr = ((const T*)a.drow)[st];
  const T inv = !in || sum == T(0) ? T(0) : T(1) / sum;
  const T* Kb = (const T*)a.k + k.b * a.sk.b + k.kh * a.sk.h;
  const T* Vb = (const T*)a.v + k.b * a.sv.b + k.kh * a.sv.h;
  Rows<T, KT, DP, VEC> fk, fv;
  if constexpr (VEC) {
    fk.start(a.sk.t, D);
    fv.start(a.sv.t, D);
  }
  auto fetch = [&](int j0) {
    fk.fetch(Kb + j0 * a.sk.t, a.sk.t, hi - j0, D);
    fv.fetch(Vb + j0 * a.sv.t, a.sv.t, hi - j0, D);
  };
  const T sl2 = (T)(a.scale * 1.4426950408889634);
  AT dq[N];
#pragma unroll
  for (int t = 0; t < N; ++t) dq[t] = AT(0);
  const bool busy = r0 < R;
  if (lo < hi) {
    fetch(lo);
    fk.put(Ks);
    fv.put(Vs);
  }
  __syncthreads();
  for (int j0 = lo; j0 < hi; j0 += KT) {
    const bool more = j0 + KT < hi;
    if (more) fetch(j0 + KT);
    if (busy) {
      typename M::vec_t xk[NF], xv[NF];
      T kc[4][N];
      lds_slice<T, DP>(xk, Ks, 0, g, c);
      lds_slice<T, DP>(xv, Vs, 0, g, c);
#pragma unroll
      for (int kt = 0; kt < KT / 16; ++kt) {
        AT s, dp, ds;
        mul_slices<T, NF>(s, xk, qf, dp, xv, gf);
        phase<T>();
        lds_cols<T, DP>(kc, Ks, 16 * kt, g, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool on = inv != T(0) && (more || j0 + 16 * kt + M::row(i, g) < hi);
          const T d = M::ex2(s[i] * sl2 - m) * inv * (dp[i] - dr);
          ds[i] = on ? d : T(0);
        }
        mul_cols<T, N>(dq, kc, ds);
        phase<T>();
        if (kt + 1 < KT / 16) {
          lds_slice<T, DP>(xk, Ks, 16 * (kt + 1), g, c);
          lds_slice<T, DP>(xv, Vs, 16 * (kt + 1), g, c);
        }
      }
    }
    __syncthreads();
    if (more) {
      fk.put(Ks);
      fv.put(Vs);
    }
    __syncthreads();
  }
  if (!in) return;
  none_without<T, N>(dq, inv);
  if (a.nsplit > 1) {
    const int64_t at = ((k.b * a.Hk + k.kh) * a.nsplit + k.split) * a.R + r;
    put_row<T, DP>((T*)a.po + at * DP, dq, (T)a.scale, DP, g, true);
  } else {
    put_row<T, DP>(group_of<T>(a, a.dq, a.sdq, k.b, k.kh) + row_at(a, a.sdq, r), dq, (T)a.scale, D, g, VEC);
  }
}

// dK and dV: a wave owns 16 keys and loops over the rows of its part. Bound by
// the MFMAs (four products): float32, 32 x 12 heads x 1024 x 2048 x 64, 124
// TFLOP/s; 8 x 12 x 1024 x 512: 232 us, 111, its 768 blocks all at once, three waves
// per SIMD; float64 591 us, 44, one wave per SIMD.
template <typename T, int DP, bool VEC>
__global__ void __launch_bounds__(256, x_waves<T>(DP, true)) xattn_bwd_kv_kernel(XArgs a) {
  using M = XM<T>;
  typedef typename M::acc_t AT;
  constexpr int N = DP / 16, LD = DP + M::PAD, QT = kKeys, NF = DP / (4 * M::VEC);
  __shared__ __attribute__((aligned(16))) T Qs[QT * LD], Gs[QT * LD];
  __shared__ __attribute__((aligned(16))) T sm[QT], si[QT], sr[QT];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15, D = (int)a.D;
  const XBlock k = x_block(a);
  const int len = (int)key_count(a, k.b), R = (int)a.R;
  // a block past the sequence's keys has only zeros to write
  const bool any = k.tile * 64 < len;
  int lo, hi;
  k.part(a.per, R, lo, hi);
  const int j0 = (k.tile * 4 + w) * 16, j = j0 + c;
  const bool in = j < len;
  const T* Kb = (const T*)a.k + k.b * a.sk.b + k.kh * a.sk.h;
  const T* Vb = (const T*)a.v + k.b * a.sv.b + k.kh * a.sv.h;
  typename M::vec_t kf[NF], vf[NF];
  load_slice<T, DP>(kf, Kb + (int64_t)(in ? j : 0) * a.sk.t, in, D, g, VEC);
  load_slice<T, DP>(vf, Vb + (int64_t)(in ? j : 0) * a.sv.t, in, D, g, VEC);
  const T* Qb = group_of<const T>(a, a.q, a.sq, k.b, k.kh);
  const T* Gb = group_of<const T>(a, a.dO, a.sdo, k.b, k.kh);
  const int64_t stats = stat_at(a, k.b, k.kh, 0);
  Rows<T, QT, DP, VEC> fq, fg;
  T nm = T(0), ni = T(0), nr = T(0);
  auto fetch = [&](int r0) {
    fq.gather([&](int r) { return r0 + r < hi ? Qb + row_at(a, a.sq, r0 + r) : nullptr; }, D);
    fg.gather([&](int r) { return r0 + r < hi ? Gb + row_at(a, a.sdo, r0 + r) : nullptr; }, D);
    if (threadIdx.x < QT) {
      const bool there = r0 + (int)threadIdx.x < hi;
      const int64_t at = stats + (there ? r0 + (int)threadIdx.x : 0);
      const T sum = there ? ((const T*)a.rowsum)[at] : T(0);
      nm = ((const T*)a.rowmax)[at];
      ni = sum == T(0) ? T(0) : T(1) / sum;
      nr = ((const T*)a.drow)[at];
    }
  };
  auto put = [&] {
    fq.put(Qs);
    fg.put(Gs);
    if (threadIdx.x < QT) {
      sm[threadIdx.x] = nm;
      si[threadIdx.x] = ni;
      sr[threadIdx.x] = nr;
    }
  };
  const T sl2 = (T)(a.scale * 1.4426950408889634);
  AT dk[N], dv[N];
#pragma unroll
  for (int t = 0; t < N; ++t) dk[t] = dv[t] = AT(0);
  const T* dsp = (const T*)a.ds + ((k.b * a.Hk + k.kh) * a.rt * a.kt + (j0 >> 4)) * 256;
  const bool busy = j0 < len;
  if (any && lo < hi) {
    fetch(lo);
    put();
  }
  __syncthreads();
  for (int r0 = lo; any && r0 < hi; r0 += QT) {
    const bool more = r0 + QT < hi;
    // A row without a finite score passes nothing on: its products with 0 would,
    // where it is infinite. (Every wave finds the same. The index is taken as new so
    // that nothing of this is kept in registers over the loop.)
    if (__any(si[lane % QT] == T(0))) {
      int f = threadIdx.x;
      asm volatile("" : "+v"(f));
#pragma unroll 1
      for (; f < QT * DP; f += 256)
        if (si[f / DP] == T(0)) Qs[f / DP * LD + f % DP] = Gs[f / DP * LD + f % DP] = T(0);
      __syncthreads();
    }
    if (more) fetch(r0 + QT);
    if (busy) {
      typename M::vec_t xq[NF], xg[NF];
      T qc[4][N], gc[4][N];
      lds_slice<T, DP>(xq, Qs, 0, g, c);
      lds_slice<T, DP>(xg, Gs, 0, g, c);
#pragma unroll
      for (int qt = 0; qt < QT / 16; ++qt) {
        T m[4], inv[4], dr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = 16 * qt + M::row(i, g);
          m[i] = sm[r];
          inv[i] = si[r];
          dr[i] = sr[r];
        }
        AT s, dp, p, ds;
        mul_slices<T, NF>(s, xq, kf, dp, xg, vf);
        phase<T>();
        lds_cols<T, DP>(gc, Gs, 16 * qt, g, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool on = in && inv[i] != T(0);
          const T e = M::ex2(s[i] * sl2 - m[i]) * inv[i], d = e * (dp[i] - dr[i]);
          p[i] = on ? e : T(0);
          ds[i] = on ? d : T(0);
        }
        // (an empty buffer where dS is not kept: no branch)
        const Rsrc tile = make_rsrc(dsp + (int64_t)((r0 >> 4) + qt) * a.kt * 256, a.ds ? 256 * sizeof(T) : 0);
        typedef int i4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < 4; i += M::VEC) {
          typename M::vec_t y;
#pragma unroll
          for (int e = 0; e < M::VEC; ++e) y[e] = ds[i + e];
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i4, y), tile, (c * 16 + 4 * g + i) * (int)sizeof(T), 0, 0);
        }
        mul_cols<T, N>(dv, gc, p);
        phase<T>();
        lds_cols<T, DP>(qc, Qs, 16 * qt, g, c);
        mul_cols<T, N>(dk, qc, ds);
        phase<T>();
        if (qt + 1 < QT / 16) {
          lds_slice<T, DP>(xq, Qs, 16 * (qt + 1), g, c);
          lds_slice<T, DP>(xg, Gs, 16 * (qt + 1), g, c);
        }
      }
    }
    __syncthreads();
    if (more) put();
    __syncthreads();
  }
  if (j >= a.Tk) return;
  if (len == 1)  // dS is 0
#pragma unroll
    for (int t = 0; t < N; ++t) dk[t] = AT(0);
  if (a.nsplit > 1) {
    const int64_t at = ((k.b * a.Hk + k.kh) * a.nsplit + k.split) * a.Tk + j;
    put_row<T, DP>((T*)a.po + at * DP, dk, (T)a.scale, DP, g, true);
    put_row<T, DP>((T*)a.pm + at * DP, dv, T(1), DP, g, true);
  } else {
    put_row<T, DP>((T*)a.dk + k.b * a.sdk.b + k.kh * a.sdk.h + (int64_t)j * a.sdk.t, dk, (T)a.scale, D, g, VEC);
    put_row<T, DP>((T*)a.dv + k.b * a.sdv.b + k.kh * a.sdv.h + (int64_t)j * a.sdv.t, dv, T(1), D, g, VEC);
  }
}

// dQ from the dS that the dK/dV pass left: one product, bound by reading dS
// (8 x 12 heads x 1024 x 512 x 64 float32, 201 MB: 66 us; float64 125).
template <typename T, int DP, bool VEC>
__global__ void __launch_bounds__(256, x_waves<T>(DP)) xattn_bwd_ds_kernel(XArgs a) {
  using M = XM<T>;
  typedef typename M::acc_t AT;
  constexpr int N = DP / 16, LD = DP + M::PAD, KT = kKeys;
  __shared__ __attribute__((aligned(16))) T Ks[KT * LD];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15, D = (int)a.D;
  const XBlock k = x_block(a);
  const int len = (int)key_count(a, k.b);
  int lo, hi;
  if (!k.part(keys_per_part(a), len, lo, hi)) return;
  if (len == 1) hi = lo;  // dS is 0
  const int r0 = (k.tile * 4 + w) * 16, R = (int)a.R, r = r0 + c;
  const bool busy = r0 < R;
  // lane (g, c): keys row(i, g) of row c, which stands where its writer's registers put it
  const int cp = M::row(1, 0) == 1 ? c : 4 * (c & 3) + (c >> 2);
  const T* dsp = (const T*)a.ds + ((k.b * a.Hk + k.kh) * a.rt + (busy ? r0 >> 4 : 0)) * a.kt * 256 + cp;
  const T* Kb = (const T*)a.k + k.b * a.sk.b + k.kh * a.sk.h;
  Rows<T, KT, DP, VEC> fk;
  if constexpr (VEC) fk.start(a.sk.t, D);
  T nx[2][4];
  auto fetch = [&](int j0) {
    fk.fetch(Kb + j0 * a.sk.t, a.sk.t, hi - j0, D);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int kt = (j0 >> 4) + s;  // a tile of keys past the sequence was not written
#pragma unroll
      for (int i = 0; i < 4; ++i)
        nx[s][i] = j0 + 16 * s < hi ? dsp[(int64_t)kt * 256 + M::row(i, g) * 16] : T(0);
    }
  };
  AT dq[N];
#pragma unroll
  for (int t = 0; t < N; ++t) dq[t] = AT(0);
  if (lo < hi) {
    fetch(lo);
    fk.put(Ks);
  }
  __syncthreads();
  for (int j0 = lo; j0 < hi; j0 += KT) {
    const bool more = j0 + KT < hi;
    AT ds[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) ds[s][i] = nx[s][i];
    if (more) fetch(j0 + KT);
    if (busy)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        T kc[4][N];
        lds_cols<T, DP>(kc, Ks, 16 * s, g, c);
        mul_cols<T, N>(dq, kc, ds[s]);
      }
    __syncthreads();
    if (more) fk.put(Ks);
    __syncthreads();
  }
  if (r >= R) return;
  none_without<T, N>(dq, ((const T*)a.rowsum)[stat_at(a, k.b, k.kh, r)]);
  if (a.nsplit > 1) {
    const int64_t at = ((k.b * a.Hk + k.kh) * a.nsplit + k.split) * a.R + r;
    put_row<T, DP>((T*)a.po + at * DP, dq, (T)a.scale, DP, g, true);
  } else {
    put_row<T, DP>(group_of<T>(a, a.dq, a.sdq, k.b, k.kh) + row_at(a, a.sdq, r), dq, (T)a.scale, D, g, VEC);
  }
}

// Sums the parts of dQ (rows: the group's) or of dK and dV (blockIdx.y 0, 1; rows:
// keys): launch and one round of loads (4 x 8 / 2 heads x 333 x 777 x 72: 12 us each).
template <typename T, int DP, bool KV>
__global__ void __launch_bounds__(256) xattn_sum_kernel(XArgs a) {
  const int64_t rows = KV ? a.Tk : a.R, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t d = id % DP, r = id / DP % rows, bh = id / DP / rows;
  // (every lane stays for the sum over lengths)
  const int64_t b = bh < a.B * a.Hk ? bh / a.Hk : 0, kh = bh % a.Hk;
  const T* p = (const T*)(KV && blockIdx.y ? a.pm : a.po) + (bh * a.nsplit * rows + r) * DP + d;
  const int n = KV ? a.nsplit : part_count(a, b);
  if (bh >= a.B * a.Hk || d >= a.D) return;
  T s = T(0);
  for (int i = 0; i < n; i += 8) {  // eight parts' loads in flight
    T x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) x[u] = p[(int64_t)(i + u < n ? i + u : n - 1) * rows * DP];
#pragma unroll
    for (int u = 0; u < 8; ++u) s = i + u < n ? s + x[u] : s;
  }
  if constexpr (KV) {
    if (blockIdx.y)
      ((T*)a.dv)[b * a.sdv.b + kh * a.sdv.h + r * a.sdv.t + d] = s;
    else
      ((T*)a.dk)[b * a.sdk.b + kh * a.sdk.h + r * a.sdk.t + d] = s;
  } else {
    group_of<T>(a, a.dq, a.sdq, b, kh)[row_at(a, a.sdq, (int)r) + d] = s;
  }
}

// Blocks along the owned axis, `per_block` of it each, and the parts of the loop
// over `loop` positions: more than one where the card would have fewer than
// `per_cu` blocks per CU, of at least two steps each, at most 64; with lengths up to
// `ragged` times as many, of which a block finds by the lengths how many are used.
// per_cu 3 (2 for up to 16 rows) was taken from sweeps of 1, 2, 3, 5: backward of
// 4 x 8 / 2 heads x 333 x 777 x 72, padded, 155 / 115 / 100 / 107 us (in 96 columns,
// as 65 to 96 then were), of 2 x 12 x 300 x 257 x 64 51 / 48 / 47 / 47; one query of 8 x 16 / 4 heads x 4999 x 128
// 39 / 34 / 44 / 41.
static int plan(XArgs& a, int64_t owned, int per_block, int64_t loop, int per_cu, int step, int ragged) {
  const int64_t tiles = cdiv(owned, per_block), blocks = a.B * a.Hk * tiles, want = per_cu * (int64_t)num_cus();
  int64_t s = blocks >= want ? 1 : cdiv(want, blocks);
  if (a.lengths && s > 1) s *= ragged;
  if (s > loop / (2 * step)) s = loop / (2 * step);
  s = s < 1 ? 1 : s > 64 ? 64 : s;
  a.step = step;
  a.per = (int)(cdiv(cdiv(loop > 0 ? loop : 1, s), step) * step);
  a.nsplit = loop > 0 ? (int)cdiv(loop, a.per) : 1;
  a.parts = (int)cdiv(want, a.Hk * tiles);
  DTMI_CHECK(tiles <= 0x7fffffff && blocks * a.nsplit <= 0x7fffffff, "cross attention: too many elements");
  a.ntile = (int)tiles;
  return DTMI_OK;
}

#define X_LAUNCH(KERNEL)                                                        \
  {                                                                             \
    const unsigned grid = (unsigned)(a.B * a.Hk * a.nsplit * a.ntile);          \
    if (a.vec)                                                                  \
      KERNEL<T, DP, true><<<grid, 256, 0, stream()>>>(a);                       \
    else                                                                        \
      KERNEL<T, DP, false><<<grid, 256, 0, stream()>>>(a);                      \
  }

template <typename T, int DP>
static int x_fwd(XArgs& a) {
  const bool few = a.R <= 16;
  if (int rc = few ? plan(a, a.R, 16, a.Tk, 2, 64, 4) : plan(a, a.R, 64, a.Tk, 3, kKeys, 4)) return rc;
  void* ws = nullptr;
  if (a.nsplit > 1) {
    const size_t n = (size_t)a.B * a.Hk * a.nsplit * a.R;
    if (int rc = pool_alloc(&ws, n * (DP + 2) * sizeof(T))) return rc;
    a.po = ws;
    a.pm = (T*)ws + n * DP;
    a.pl = (T*)a.pm + n;
  }
  if (few)
    X_LAUNCH(xattn_rows_kernel)
  else
    X_LAUNCH(xattn_fwd_kernel)
  if (a.nsplit > 1) {
    const int64_t rows = a.B * a.Hk * a.R;
    if (rows <= 2048)
      xattn_join_few_kernel<T, DP><<<(unsigned)rows, 256, 0, stream()>>>(a);
    else
      xattn_join_kernel<T, DP><<<(unsigned)cdiv(rows, 4), 256, 0, stream()>>>(a);
  }
  const hipError_t e = hipGetLastError();
  if (ws) pool_free(ws);
  return e == hipSuccess ? DTMI_OK : fail_hip(e, "dtmi_xattn_fwd", __FILE__, __LINE__);
}

template <typename T, int DP>
static int x_bwd_kv(XArgs& a) {
  if (int rc = plan(a, a.Tk, 64, a.R, 3, kKeys, 1)) return rc;
  void* ws = nullptr;
  if (a.nsplit > 1) {
    const size_t n = (size_t)a.B * a.Hk * a.nsplit * a.Tk * DP;
    if (int rc = pool_alloc(&ws, 2 * n * sizeof(T))) return rc;
    a.po = ws;
    a.pm = (T*)ws + n;
  }
  X_LAUNCH(xattn_bwd_kv_kernel)
  if (a.nsplit > 1)
    xattn_sum_kernel<T, DP, true>
        <<<dim3((unsigned)cdiv(a.B * a.Hk * a.Tk * DP, 256), 2), 256, 0, stream()>>>(a);
  const hipError_t e = hipGetLastError();
  if (ws) pool_free(ws);
  return e == hipSuccess ? DTMI_OK : fail_hip(e, "dtmi_xattn_bwd: dK, dV", __FILE__, __LINE__);
}

template <typename T, int DP>
static int x_bwd_q(XArgs& a) {
  if (int rc = plan(a, a.R, 64, a.Tk, 3, kKeys, 4)) return rc;
  void* ws = nullptr;
  if (a.nsplit > 1) {
    if (int rc = pool_alloc(&ws, (size_t)a.B * a.Hk * a.nsplit * a.R * DP * sizeof(T))) return rc;
    a.po = ws;
  }
  if (a.ds)
    X_LAUNCH(xattn_bwd_ds_kernel)
  else
    X_LAUNCH(xattn_bwd_q_kernel)
  if (a.nsplit > 1)
    xattn_sum_kernel<T, DP, false><<<(unsigned)cdiv(a.B * a.Hk * a.R * DP, 256), 256, 0, stream()>>>(a);
  const hipError_t e = hipGetLastError();
  if (ws) pool_free(ws);
  return e == hipSuccess ? DTMI_OK : fail_hip(e, "dtmi_xattn_bwd: dQ", __FILE__, __LINE__);
}
#undef X_LAUNCH

template <typename T, int DP>
static int x_bwd(XArgs& a) {
  void* dr = nullptr;
  if (int rc = pool_alloc(&dr, (size_t)a.B * a.H * a.Tq * sizeof(T))) return rc;
  a.drow = dr;
  xattn_drow_kernel<T><<<(unsigned)cdiv(a.B * a.Hk * a.R, 16), 256, 0, stream()>>>(a);
  const hipError_t e = hipGetLastError();
  int rc = e == hipSuccess ? DTMI_OK : fail_hip(e, "dtmi_xattn_bwd: row dots", __FILE__, __LINE__);
  // dS handed from the one pass to the other, where it may be kept: 8 bytes of
  // traffic per score (float32) against two of the three products that the dQ pass
  // would take. Backward of 8 x 12 heads x 1024 queries, us without and with: 512
  // keys x 32 237 / 195, 512 x 64 400 / 312, 2048 x 32 824 / 697, 2048 x 64 1492 / 1127.
  a.rt = cdiv(a.R, kKeys) * (kKeys / 16);
  a.kt = cdiv(a.Tk, 16);
  const int64_t bytes = a.B * a.Hk * a.rt * a.kt * 256 * (int64_t)sizeof(T);
  if (rc == DTMI_OK && bytes <= ds_limit() && pool_alloc(&a.ds, bytes) != DTMI_OK) a.ds = nullptr;
  if (rc == DTMI_OK) rc = x_bwd_kv<T, DP>(a);
  if (rc == DTMI_OK) rc = x_bwd_q<T, DP>(a);
  if (a.ds) pool_free(a.ds);
  pool_free(dr);
  return rc;
}

// Columns that a head is padded to. 48 and 80 beside the multiples of 32: forward /
// backward of 8 x 12 heads x 1024 x 512 x 40 124 / 304 us in 64 columns, 105 / 253
// in 48; x 72 188 / 510 in 96, 154 / 440 in 80.
template <typename T>
static int x_dispatch(XArgs& a, bool bwd) {
  if (a.D <= 32) return bwd ? x_bwd<T, 32>(a) : x_fwd<T, 32>(a);
  if (a.D <= 48) return bwd ? x_bwd<T, 48>(a) : x_fwd<T, 48>(a);
  if (a.D <= 64) return bwd ? x_bwd<T, 64>(a) : x_fwd<T, 64>(a);
  if (a.D <= 80) return bwd ? x_bwd<T, 80>(a) : x_fwd<T, 80>(a);
  if (a.D <= 96) return bwd ? x_bwd<T, 96>(a) : x_fwd<T, 96>(a);
  return bwd ? x_bwd<T, 128>(a) : x_fwd<T, 128>(a);
}

static int x_shape(const char* what, int dtype, int64_t B, int64_t H, int64_t Hk, int64_t Tq, int64_t Tk, int64_t D) {
  DTMI_CHECK(dtype == DTMI_F32 || dtype == DTMI_F64, "%s: dtype must be DTMI_F32 or DTMI_F64 (got %d)", what, dtype);
  DTMI_CHECK(B >= 0 && H >= 0 && Tq >= 0 && Tk >= 0, "%s: negative size", what);
  DTMI_CHECK(Hk >= 1 && H % Hk == 0, "%s: %lld heads do not share %lld key/value heads", what, (long long)H,
             (long long)Hk);
  DTMI_CHECK(D >= 1 && D <= 128, "%s: head dimension 1 to 128 (got %lld)", what, (long long)D);
  DTMI_CHECK(Tk < ((int64_t)1 << 31) - 4096, "%s: too many keys", what);
  DTMI_CHECK(B * H * Tq < ((int64_t)1 << 31) - 4096 && B * Hk * Tk * 128 < ((int64_t)1 << 38), "%s: too many elements", what);
  return DTMI_OK;
}

static HT ht(const int64_t* s) { return s ? HT{s[0], s[1], s[2]} : HT{0, 0, 0}; }
template <typename T>
static bool x_vec(const void* p, const HT& s) {
  constexpr int V = 16 / sizeof(T);
  return aligned(p, 16) && s.b % V == 0 && s.h % V == 0 && s.t % V == 0 && s.t >= 0 && s.t < (1 << 23);
}

template <typename T>
static int x_zero_rows(void* p, const HT& s, int64_t B, int64_t H, int64_t T_, int64_t D) {
  const int64_t shape[4] = {B, H, T_, D}, to[4] = {s.b, s.h, s.t, 1}, from[4] = {0, 0, 0, 0};
  void* zero = nullptr;
  if (int rc = pool_alloc(&zero, sizeof(T))) return rc;
  const int dt = sizeof(T) == 4 ? DTMI_F32 : DTMI_F64;
  int rc = dtmi_fill(dt, zero, 0.0, 1);
  if (rc == DTMI_OK) rc = dtmi_copy_strided(dt, p, to, zero, from, 4, shape);
  pool_free(zero);
  return rc;
}

template <typename T>
static int xattn_fwd(XArgs& a) {
  a.vec = a.D % (16 / sizeof(T)) == 0 && x_vec<T>(a.q, a.sq) && x_vec<T>(a.k, a.sk) && x_vec<T>(a.v, a.sv) &&
          x_vec<T>(a.out, a.so);
  return x_dispatch<T>(a, false);
}
template <typename T>
static int xattn_bwd(XArgs& a) {
  if (a.R == 0 || a.Tk == 0) {
    int rc = DTMI_OK;
    if (a.R > 0) rc = x_zero_rows<T>(a.dq, a.sdq, a.B, a.H, a.Tq, a.D);
    if (rc == DTMI_OK && a.Tk > 0) rc = x_zero_rows<T>(a.dk, a.sdk, a.B, a.Hk, a.Tk, a.D);
    if (rc == DTMI_OK && a.Tk > 0) rc = x_zero_rows<T>(a.dv, a.sdv, a.B, a.Hk, a.Tk, a.D);
    return rc;
  }
  a.vec = a.D % (16 / sizeof(T)) == 0 && x_vec<T>(a.q, a.sq) && x_vec<T>(a.k, a.sk) && x_vec<T>(a.v, a.sv) &&
          x_vec<T>(a.dO, a.sdo) && x_vec<T>(a.dq, a.sdq) && x_vec<T>(a.dk, a.sdk) && x_vec<T>(a.dv, a.sdv);
  return x_dispatch<T>(a, true);
}

}  // namespace dtmi

using namespace dtmi;

DTMI_EXPORT int dtmi_xattn_fwd(int dtype, int64_t B, int64_t H, int64_t Hk, int64_t Tq, int64_t Tk, int64_t D,
                               double scale, const void* q, const int64_t* q_strides, const void* k,
                               const int64_t* k_strides, const void* v, const int64_t* v_strides,
                               const int64_t* lengths, void* o, const int64_t* o_strides, void* rowmax, void* rowsum) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  if (int rc = x_shape("dtmi_xattn_fwd", dtype, B, H, Hk, Tq, Tk, D)) return rc;
  if (B == 0 || H == 0 || Tq == 0) return DTMI_OK;
  DTMI_CHECK(q && o && q_strides && o_strides && (Tk == 0 || (k && v && k_strides && v_strides)) && !rowmax == !rowsum,
             "dtmi_xattn_fwd: NULL operand");
  XArgs a{};
  a.q = q, a.k = k, a.v = v, a.out = o, a.lengths = lengths, a.rowmax = rowmax, a.rowsum = rowsum;
  a.sq = ht(q_strides), a.sk = ht(k_strides), a.sv = ht(v_strides), a.so = ht(o_strides);
  a.B = B, a.H = H, a.Hk = Hk, a.Tq = Tq, a.Tk = Tk, a.D = D, a.G = H / Hk, a.R = a.G * Tq, a.scale = scale;
  a.by_tq = FastDiv((uint32_t)(a.R > 0 ? Tq : 1));
  TimedLaunch tl(DTMI_FAM_OTHER, 4.0 * B * H * Tq * Tk * D);
  return dtype == DTMI_F32 ? xattn_fwd<float>(a) : xattn_fwd<double>(a);
  DTMI_BODY_END
}

DTMI_EXPORT int dtmi_xattn_bwd(int dtype, int64_t B, int64_t H, int64_t Hk, int64_t Tq, int64_t Tk, int64_t D,
                               double scale, const void* q, const int64_t* q_strides, const void* k,
                               const int64_t* k_strides, const void* v, const int64_t* v_strides,
                               const int64_t* lengths, const void* o, const int64_t* o_strides, const void* dO,
                               const int64_t* dO_strides, const void* rowmax, const void* rowsum, void* dq,
                               const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                               const int64_t* dv_strides) {
  DTMI_BODY_BEGIN
  DTMI_REQUIRE_INIT();
  if (int rc = x_shape("dtmi_xattn_bwd", dtype, B, H, Hk, Tq, Tk, D)) return rc;
  if (B == 0) return DTMI_OK;
  DTMI_CHECK((H == 0 || Tq == 0 || (q && o && dO && dq && rowmax && rowsum && q_strides && o_strides && dO_strides && dq_strides)) &&
                 (Tk == 0 || (k && v && dk && dv && k_strides && v_strides && dk_strides && dv_strides)),
             "dtmi_xattn_bwd: NULL operand");
  XArgs a{};
  a.q = q, a.k = k, a.v = v, a.o = o, a.dO = dO, a.dq = dq, a.dk = dk, a.dv = dv, a.lengths = lengths;
  a.rowmax = const_cast<void*>(rowmax), a.rowsum = const_cast<void*>(rowsum);
  a.sq = ht(q_strides), a.sk = ht(k_strides), a.sv = ht(v_strides), a.so = ht(o_strides), a.sdo = ht(dO_strides);
  a.sdq = ht(dq_strides), a.sdk = ht(dk_strides), a.sdv = ht(dv_strides);
  a.B = B, a.H = H, a.Hk = Hk, a.Tq = Tq, a.Tk = Tk, a.D = D, a.G = H / Hk, a.R = a.G * Tq, a.scale = scale;
  a.by_tq = FastDiv((uint32_t)(a.R > 0 ? Tq : 1));
  TimedLaunch tl(DTMI_FAM_OTHER, 14.0 * B * H * Tq * Tk * D);
  return dtype == DTMI_F32 ? xattn_bwd<float>(a) : xattn_bwd<double>(a);
  DTMI_BODY_END
}
