// The residual sum between two sub-layers' norms on the flat node layout:
//   rows'  = rows + s * act(z) * (g_p * norm(u) + b_p)
//   normed = g_n * norm(rows') + b_n
// with norm the merged equivariant normalisation (frequency 0 centred, one
// denominator sqrt(sum_k w_k c_k^2 + eps) pooled over the frequencies'
// mean squares: w = 1 / (a0 present) on frequency 0 and 1 / (2 m present) on a
// frequency of m copies), act(z) = factor sigmoid(z) one gate a copy, s one
// scale a coordinate.  Without g_p the branch is not normalised, without g_n
// nothing is normalised behind the sum, without z or s the factor is one.
// The next norm reads the sum before it is rounded to the rows' type.
//
// Backward, from dy (of rows') and dh (of normed):
//   G  = dy + norm'(rows')^T (g_n dh)          (the gradient of rows)
//   dz = act'(z) sum over the copy of G s (g_p uhat + b_p)
//   du = norm'(u)^T (G act(z) s g_p)
// and the per-coordinate sums over the rows A = sum G act uhat, B = sum G act,
// C = sum dh xhat, E = sum dh, of which the parameters' gradients are made:
// dg_p = s A, ds = g_p A + b_p B, db_p = s B, dg_n = C, db_n = E.  rows' is
// formed again from rows, u and z, which the pass reads anyway: what rounding
// the stored rows' to bfloat16 loses would otherwise enter C and the rows'
// gradient.
//
// One pass over the data each way, so the bytes bound it: 524,288 rows of 160 in
// float with gates take 301 us forward (5.1 TB/s) and 511 backward (4.75), 262,144
// bfloat16 rows with a float branch 95 and 213 (the latter at 3.6 TB/s: its registers
// leave two waves a SIMD).  A row's units (16
// bytes of float or double, 8 of bfloat16, or one copy where a multiplicity, a
// pointer or the gates' rows are not whole units) are shared by 2^k lanes with at most
// kMaxUnits<...> units a lane, all in registers; the norms' sums are shuffles
// within those lanes; a wave holds 64 / 2^k rows.  Coefficients sit in LDS, since
// each lane would otherwise hold five registers of them for every number of a row;
// a workgroup makes them from the parameters as the modules hold them, so a call
// is one launch forward and two backward.  The waves are persistent; the backward's
// sums stay in registers over a wave's rows, are added over the workgroup in a fixed order,
// and a second kernel adds the workgroups' rows in a fixed order (no atomics).
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace gm {
namespace {

constexpr int kRnMaxFreq = 8;           // nonzero frequencies
constexpr int kRnSlots = kRnMaxFreq + 1;  // frequency 0, then the nonzero ones
constexpr int kRnThreads = 256;
constexpr int kRnWaves = kRnThreads / kWave;
// The backward's workgroups: eight waves where their registers let a CU hold eight (half as many rows of sums to add
// as with four: that kernel 17 -> 10 us), four above that.
template <typename X, bool kCopies, int NS>
constexpr int kRnBackThreads = NS <= (kCopies ? 4 : (sizeof(X) == 8 ? 2 : 3)) && sizeof(X) * NS <= 16 ? 512 : 256;
constexpr int kRnMaxWidth = 1024;

struct rbf16 {
  uint16_t bits;
};

template <typename T>
struct RnAcc {
  using type = float;
};
template <>
struct RnAcc<double> {
  using type = double;
};

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ float widen(rbf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }

// The row type's numbers, bfloat16 rounded to nearest even.
__device__ __forceinline__ void narrow(float v, float& o) { o = v; }
__device__ __forceinline__ void narrow(double v, double& o) { o = v; }
__device__ __forceinline__ void narrow(float v, rbf16& o) {
  const __bf16 b = static_cast<__bf16>(v);
  __builtin_memcpy(&o.bits, &b, 2);
}

// V consecutive numbers of type T at p as one load or store of up to 16 bytes each; bfloat16 ones as 32-bit words.
template <typename T, int V>
struct alignas(sizeof(T) * V >= 16 ? 16 : sizeof(T) * V) Pack {
  T v[V];
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
template <int V>
__device__ __forceinline__ void load_n(const rbf16* p, float (&out)[V]) {
  static_assert(V == 2 || V == 4, "whole words");
  uint32_t w[V / 2];
  if constexpr (V == 4) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    out[2 * i] = __uint_as_float(w[i] << 16);
    out[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <int V>
__device__ __forceinline__ void store_n(rbf16* p, const float (&in)[V]) {
  static_assert(V == 2 || V == 4, "whole words");
  uint32_t w[V / 2];
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const bf16x2 b = {static_cast<__bf16>(in[2 * i]), static_cast<__bf16>(in[2 * i + 1])};
    w[i] = __builtin_bit_cast(uint32_t, b);
  }
  if constexpr (V == 4)
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t*>(p) = w[0];
}
template <int V, typename T, typename A>
__device__ __forceinline__ void load_n(const T* p, A (&out)[V]) {
  const Pack<T, V> x = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = widen(x.v[i]);
}
template <int V, typename T, typename A>
__device__ __forceinline__ void store_n(T* p, const A (&in)[V]) {
  Pack<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) narrow(in[i], x.v[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = x;
}

template <typename X, typename U>
struct RnArgs {
  using A = typename RnAcc<X>::type;
  int64_t n_rows;
  int D, a0, copies, present, nf;
  int off[kRnMaxFreq], mult[kRnMaxFreq];
  int units, scalar_units;  // a row's units, the first of them frequency 0's
  int lanes, shift;         // lanes a row (a power of two), its logarithm
  const X* x;
  const U* u;
  const X* z;           // (n_rows, copies) or null
  // the parameters as the modules hold them: a vector a frequency, one number a copy
  const A* gain[kRnSlots];       // where normalise
  const A* scale[kRnSlots];      // where scaled
  const A* next_gain[kRnSlots];  // where next
  const A* offset;               // (a0) or null
  const A* next_offset;          // (a0) or null
  bool normalise, scaled, next;  // the branch is normalised, its copies scaled, the sum normalised
  A factor, eps, next_eps;
  X* y;
  X* normed;
  A* stats;  // (n_rows, 4): the branch's mean and 1 / d, the sum's
  // backward
  const X* dy;  // or null
  const X* dn;  // or null
  X* dx;
  U* du;
  X* dz;
  A* partial;  // (workgroups, 4, units V)
  A* dparams;  // dgain (copies), doffset (a0), dscale (copies), dnext_gain (copies), dnext_offset (a0)
};

// Where coordinate k sits: its frequency's slot, its copy among that frequency's, that frequency's copies.
struct RnPlace {
  int slot, copy, mult;
};
template <typename Args>
__device__ __forceinline__ RnPlace place_of(const Args& a, int k) {
  if (k < a.a0) return {0, k, a.a0};
  int f = 0;
  for (int g = 1; g < a.nf; ++g)
    if (k >= a.off[g]) f = g;
  return {1 + f, (k - a.off[f]) / 2, a.mult[f]};
}

// What a row's unit is.  Units: V numbers of one kind (scalars, or whole pairs), their gates V or V / 2 numbers; four
// of bfloat16 too (eight a unit leave a lane 24 numbers of each row and the backward one wave a SIMD).  Copies
// (kCopies): one copy, of one or two numbers, V = 2.
template <typename X, typename U, bool kCopies>
struct RnUnit {
  using A = typename RnAcc<X>::type;
  using Args = RnArgs<X, U>;
  static constexpr int V = kCopies || sizeof(X) == 8 ? 2 : 4;
  static __device__ __forceinline__ int first(const Args& a, int unit) {
    if constexpr (kCopies)
      return unit < a.a0 ? unit : 2 * unit - a.a0;
    else
      return unit * V;
  }
  template <typename T>
  static __device__ __forceinline__ void load(const Args& a, const T* row, int unit, A (&v)[V]) {
    const int k = first(a, unit);
    if constexpr (kCopies) {
      v[0] = widen(row[k]);
      v[1] = unit < a.a0 ? A(0) : widen(row[k + 1]);
    } else {
      load_n<V>(row + k, v);
    }
  }
  template <typename T>
  static __device__ __forceinline__ void store(const Args& a, T* row, int unit, const A (&v)[V]) {
    const int k = first(a, unit);
    if constexpr (kCopies) {
      T t;
      narrow(v[0], t);
      row[k] = t;
      if (unit >= a.a0) {
        narrow(v[1], t);
        row[k + 1] = t;
      }
    } else {
      store_n<V>(row + k, v);
    }
  }
  // the gates of a unit's numbers, a pair's given twice
  static __device__ __forceinline__ void load_gates(const Args& a, const X* row, int unit, A (&g)[V]) {
    if constexpr (kCopies) {
      g[0] = g[1] = widen(row[unit]);
    } else {
      // selects, not a branch's stores: those went through scratch for bfloat16 (510 us against 345 then for the
      // backward of 262,144 rows of 160 with a float branch, 189 against 108 for the forward)
      const bool scalar = unit < a.scalar_units;
      A lo[V / 2], hi[V / 2];
      const X* p = row + (scalar ? unit * V : (unit * V + a.a0) / 2);
      load_n<V / 2>(p, lo);
      load_n<V / 2>(scalar ? p + V / 2 : p, hi);
#pragma unroll
      for (int i = 0; i < V; ++i) g[i] = scalar ? (i < V / 2 ? lo[i] : hi[i - V / 2]) : lo[i / 2];
    }
  }
  static __device__ __forceinline__ void store_gates(const Args& a, X* row, int unit, const A (&d)[V]) {
    if constexpr (kCopies) {
      X t;
      narrow(unit < a.a0 ? d[0] : d[0] + d[1], t);
      row[unit] = t;
    } else {
      const bool scalar = unit < a.scalar_units;
      A lo[V / 2], hi[V / 2];
      X* p = row + (scalar ? unit * V : (unit * V + a.a0) / 2);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        lo[i] = scalar ? d[i] : d[2 * i] + d[2 * i + 1];
        hi[i] = d[V / 2 + i];
      }
      store_n<V / 2>(p, lo);
      if (scalar) store_n<V / 2>(p + V / 2, hi);
    }
  }
};

enum Table { kGain = 0, kOffset = 1, kNextGain = 2, kNextOffset = 3, kShare = 4, kTables = 5 };

// The coefficients of every coordinate in LDS: s g_p, s b_p, g_n, b_n, its share of the pooled mean square.
template <typename X, typename U, bool kCopies>
struct RnTables {
  using A = typename RnAcc<X>::type;
  using Args = RnArgs<X, U>;
  using Unit = RnUnit<X, U, kCopies>;
  static constexpr int V = Unit::V;
  A* lds;
  __device__ __forceinline__ void fill(const Args& a, A* shared) {
    lds = shared;
    for (int k = threadIdx.x; k < a.D; k += blockDim.x) {
      const RnPlace at = place_of(a, k);
      const A s = a.scaled ? a.scale[at.slot][at.copy] : A(1);
      lds[kGain * a.D + k] = a.normalise ? s * a.gain[at.slot][at.copy] : s;
      lds[kOffset * a.D + k] = a.offset && at.slot == 0 ? s * a.offset[k] : A(0);
      lds[kNextGain * a.D + k] = a.next ? a.next_gain[at.slot][at.copy] : A(0);
      lds[kNextOffset * a.D + k] = a.next_offset && at.slot == 0 ? a.next_offset[k] : A(0);
      lds[kShare * a.D + k] = A(1) / (A(at.slot == 0 ? 1 : 2) * A(at.mult) * A(a.present));
    }
    __syncthreads();
  }
  // a unit's numbers (zero past a scalar copy)
  __device__ __forceinline__ void get(const Args& a, int t, int unit, A (&c)[V]) const {
    const int k = Unit::first(a, unit);
    if constexpr (kCopies) {
      c[0] = lds[t * a.D + k];
      c[1] = unit < a.a0 ? A(0) : lds[t * a.D + k + 1];
    } else {
      load_n<V>(lds + t * a.D + k, c);
    }
  }
};

// Sum over a row's lanes; every lane gets it.
template <typename A>
__device__ __forceinline__ A row_sum(A v, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// A lane's j-th unit of a row: past the last one it is that one once more, loaded and not stored, its numbers zeroed
// where they would count (no branches: predicated loads waited for one another).
struct RnLane {
  int unit;
  bool on, scalar;
};
template <typename Args>
__device__ __forceinline__ RnLane lane_unit(const Args& a, int lane, int j) {
  const int unit = lane + j * a.lanes;
  return {unit < a.units ? unit : a.units - 1, unit < a.units, unit < a.scalar_units};
}

// Mean of the scalars and 1 / d of the numbers a row's lanes hold (zero past the last unit).
template <typename X, typename U, bool kCopies, int NS>
__device__ __forceinline__ void row_stats(const RnArgs<X, U>& a, const RnTables<X, U, kCopies>& tables, int lane,
                                          const typename RnAcc<X>::type (&v)[NS][RnUnit<X, U, kCopies>::V],
                                          typename RnAcc<X>::type eps, typename RnAcc<X>::type& mean,
                                          typename RnAcc<X>::type& inv_d) {
  using A = typename RnAcc<X>::type;
  constexpr int V = RnUnit<X, U, kCopies>::V;
  mean = A(0);
  if (a.a0 > 0) {
    A s = A(0);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const bool scalar = lane_unit(a, lane, j).scalar;
#pragma unroll
      for (int i = 0; i < V; ++i) s += scalar ? v[j][i] : A(0);  // a scalar copy's second number is zero
    }
    mean = row_sum(s, a.lanes) / A(a.a0);
  }
  A q = A(0);
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const RnLane at = lane_unit(a, lane, j);
    A w[V];
    tables.get(a, kShare, at.unit, w);
    const A m = at.scalar ? mean : A(0);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const A c = v[j][i] - m;
      q += w[i] * c * c;
    }
  }
  inv_d = A(1) / sqrt(row_sum(q, a.lanes) + eps);
}

// 1 / (1 + exp(-z)); in float from v_exp_f32 and v_rcp_f32, each a step off (the exponent's rounding |z| / 2 steps
// more of what exp(-z) contributes): a tenth of a call's and a division's instructions.
__device__ __forceinline__ float rn_sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * z));
}
__device__ __forceinline__ double rn_sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }
// The gates of a unit's numbers from their pre-activations; `pairs`: no lane's unit of this step is scalars, and a
// pair's two numbers share one.
template <int V, typename A>
__device__ __forceinline__ void rn_gates(A (&g)[V], bool pairs) {
  if (pairs) {
#pragma unroll
    for (int i = 0; i < V; i += 2) g[i] = g[i + 1] = rn_sigmoid(g[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = rn_sigmoid(g[i]);
  }
}

template <typename X, typename U, bool kCopies, int NS>
__global__ __launch_bounds__(kRnThreads) void residual_norm_forward_kernel(RnArgs<X, U> a) {
  using A = typename RnAcc<X>::type;
  using Unit = RnUnit<X, U, kCopies>;
  constexpr int V = Unit::V;
  extern __shared__ __align__(16) unsigned char rn_lds[];
  RnTables<X, U, kCopies> tables;
  tables.fill(a, reinterpret_cast<A*>(rn_lds));
  const int in_wave = threadIdx.x % kWave, lane = in_wave & (a.lanes - 1);
  const int per_wave = kWave >> a.shift;
  const int64_t step = (int64_t)gridDim.x * kRnWaves * per_wave;
  int64_t row = ((int64_t)blockIdx.x * kRnWaves + threadIdx.x / kWave) * per_wave + (in_wave >> a.shift);
  // whole waves take every step: the rows past the last one shadow it and store nothing
  for (int64_t at = row - (in_wave >> a.shift); at < a.n_rows; at += step, row += step) {
    const bool live = row < a.n_rows;
    const int64_t r = live ? row : a.n_rows - 1;
    A x[NS][V], u[NS][V], g[NS][V];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const RnLane at_j = lane_unit(a, lane, j);
      Unit::load(a, a.u + r * a.D, at_j.unit, u[j]);
      Unit::load(a, a.x + r * a.D, at_j.unit, x[j]);
    }
    if (a.z) {
#pragma unroll
      for (int j = 0; j < NS; ++j) Unit::load_gates(a, a.z + r * a.copies, lane_unit(a, lane, j).unit, g[j]);
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const bool on = lane_unit(a, lane, j).on;
#pragma unroll
      for (int i = 0; i < V; ++i) u[j][i] = on ? u[j][i] : A(0);
    }
    A mean = A(0), inv = A(1);
    if (a.normalise) row_stats<X, U, kCopies, NS>(a, tables, lane, u, a.eps, mean, inv);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const RnLane at_j = lane_unit(a, lane, j);
      A gain[V], offset[V];
      tables.get(a, kGain, at_j.unit, gain);
      tables.get(a, kOffset, at_j.unit, offset);
      const A m = at_j.scalar ? mean : A(0);
#pragma unroll
      for (int i = 0; i < V; ++i) u[j][i] = gain[i] * ((u[j][i] - m) * inv) + offset[i];
    }
    if (a.z) {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        rn_gates<V>(g[j], j * a.lanes >= a.scalar_units);
#pragma unroll
        for (int i = 0; i < V; ++i) u[j][i] *= a.factor * g[j][i];
      }
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const RnLane at_j = lane_unit(a, lane, j);
#pragma unroll
      for (int i = 0; i < V; ++i) x[j][i] = at_j.on ? x[j][i] + u[j][i] : A(0);
      if (kCopies && at_j.scalar) x[j][1] = A(0);
      if (live && at_j.on) Unit::store(a, a.y + r * a.D, at_j.unit, x[j]);
    }
    A mean2 = A(0), inv2 = A(1);
    if (a.next) {
      row_stats<X, U, kCopies, NS>(a, tables, lane, x, a.next_eps, mean2, inv2);
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const RnLane at_j = lane_unit(a, lane, j);
        A gain[V], offset[V], out[V];
        tables.get(a, kNextGain, at_j.unit, gain);
        tables.get(a, kNextOffset, at_j.unit, offset);
        const A m = at_j.scalar ? mean2 : A(0);
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = gain[i] * ((x[j][i] - m) * inv2) + offset[i];
        if (live && at_j.on) Unit::store(a, a.normed + r * a.D, at_j.unit, out);
      }
    }
    if (a.stats && live && lane == 0) {
      A* st = a.stats + 4 * r;
      st[0] = mean;
      st[1] = inv;
      st[2] = mean2;
      st[3] = inv2;
    }
  }
}

template <typename X, typename U, bool kCopies, int NS>
__global__ __launch_bounds__((kRnBackThreads<X, kCopies, NS>)) void residual_norm_backward_kernel(RnArgs<X, U> a) {
  using A = typename RnAcc<X>::type;
  using Unit = RnUnit<X, U, kCopies>;
  constexpr int V = Unit::V, kThreads = kRnBackThreads<X, kCopies, NS>, kWaves = kThreads / kWave;
  extern __shared__ __align__(16) unsigned char rn_lds[];
  RnTables<X, U, kCopies> tables;
  tables.fill(a, reinterpret_cast<A*>(rn_lds));
  const int in_wave = threadIdx.x % kWave, lane = in_wave & (a.lanes - 1);
  const int per_wave = kWave >> a.shift;
  const int64_t step = (int64_t)gridDim.x * kWaves * per_wave;
  const A by_scalars = a.a0 > 0 ? A(1) / A(a.a0) : A(0);
  // the sums over this lane's rows: G act uhat, G act, dn xhat, dn (the second and fourth are read of scalars only)
  A sums[4][NS][V];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) sums[t][j][i] = A(0);
  int64_t row = ((int64_t)blockIdx.x * kWaves + threadIdx.x / kWave) * per_wave + (in_wave >> a.shift);
  for (int64_t at = row - (in_wave >> a.shift); at < a.n_rows; at += step, row += step) {
    const bool live = row < a.n_rows;
    const int64_t r = live ? row : a.n_rows - 1;
    const A* st = a.stats + 4 * r;
    const A mean = st[0], inv = st[1], mean2 = st[2], inv2 = st[3];
    A uh[NS][V], G[NS][V], act[NS][V], xh[NS][V], dn[NS][V];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      Unit::load(a, a.u + r * a.D, lane_unit(a, lane, j).unit, uh[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        G[j][i] = A(0);
        act[j][i] = A(1);
      }
    }
    if (a.dn) {
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const int unit = lane_unit(a, lane, j).unit;
        Unit::load(a, a.x + r * a.D, unit, xh[j]);
        Unit::load(a, a.dn + r * a.D, unit, dn[j]);
      }
    }
    if (a.dy) {
#pragma unroll
      for (int j = 0; j < NS; ++j) Unit::load(a, a.dy + r * a.D, lane_unit(a, lane, j).unit, G[j]);
    }
    if (a.z) {
#pragma unroll
      for (int j = 0; j < NS; ++j) Unit::load_gates(a, a.z + r * a.copies, lane_unit(a, lane, j).unit, act[j]);
#pragma unroll
      for (int j = 0; j < NS; ++j) rn_gates<V>(act[j], j * a.lanes >= a.scalar_units);
    }
    const A factor = a.z ? a.factor : A(1);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const RnLane at_j = lane_unit(a, lane, j);
      const bool counts = at_j.on && live;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        uh[j][i] = at_j.on ? (uh[j][i] - (at_j.scalar ? mean : A(0))) * inv : A(0);
        G[j][i] = counts ? G[j][i] : A(0);
      }
    }
    // xhat from the sum formed again; p and m, the next norm's two sums; its part of G
    if (a.dn) {
      A p = A(0), m = A(0);
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const RnLane at_j = lane_unit(a, lane, j);
        const bool counts = at_j.on && live;
        A gain[V], offset[V], next[V];
        tables.get(a, kGain, at_j.unit, gain);
        tables.get(a, kOffset, at_j.unit, offset);
        tables.get(a, kNextGain, at_j.unit, next);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const A y = xh[j][i] + factor * act[j][i] * (gain[i] * uh[j][i] + offset[i]);
          xh[j][i] = (y - (at_j.scalar ? mean2 : A(0))) * inv2;
          dn[j][i] = counts ? dn[j][i] : A(0);
          sums[2][j][i] += dn[j][i] * xh[j][i];
          sums[3][j][i] += dn[j][i];
          dn[j][i] *= next[i];
          p += dn[j][i] * xh[j][i];
          m += at_j.scalar ? dn[j][i] : A(0);
        }
      }
      p = row_sum(p, a.lanes);
      m = row_sum(m, a.lanes) * by_scalars;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const RnLane at_j = lane_unit(a, lane, j);
        A w[V];
        tables.get(a, kShare, at_j.unit, w);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const A d = inv2 * (dn[j][i] - (at_j.scalar ? m : A(0)) - p * xh[j][i] * w[i]);
          G[j][i] += at_j.on ? d : A(0);
        }
        if (kCopies && at_j.scalar) G[j][1] = A(0);
      }
    }
    A p1 = A(0), m1 = A(0);
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const RnLane at_j = lane_unit(a, lane, j);
      A gain[V], offset[V], d[V];
      if (live && at_j.on) Unit::store(a, a.dx + r * a.D, at_j.unit, G[j]);
      tables.get(a, kGain, at_j.unit, gain);
      tables.get(a, kOffset, at_j.unit, offset);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const A s = act[j][i];
        G[j][i] *= factor * s;
        d[i] = G[j][i] * (gain[i] * uh[j][i] + offset[i]) * (A(1) - s);  // of the gate's argument
        sums[0][j][i] += G[j][i] * uh[j][i];
        sums[1][j][i] += G[j][i];
        G[j][i] *= gain[i];
        p1 += G[j][i] * uh[j][i];
        m1 += at_j.scalar ? G[j][i] : A(0);
      }
      if (a.z) {
        if (live && at_j.on) Unit::store_gates(a, a.dz + r * a.copies, at_j.unit, d);
      }
    }
    if (a.normalise) {
      p1 = row_sum(p1, a.lanes);
      m1 = row_sum(m1, a.lanes) * by_scalars;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const RnLane at_j = lane_unit(a, lane, j);
        A w[V];
        tables.get(a, kShare, at_j.unit, w);
#pragma unroll
        for (int i = 0; i < V; ++i)
          G[j][i] = inv * (G[j][i] - (at_j.scalar ? m1 : A(0)) - p1 * uh[j][i] * w[i]);
      }
    }
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      const RnLane at_j = lane_unit(a, lane, j);
      if (live && at_j.on) Unit::store(a, a.du + r * a.D, at_j.unit, G[j]);
    }
  }
  // over the wave's rows, then over the workgroup's waves in order
  A* shared = reinterpret_cast<A*>(rn_lds);
  const int width = a.units * V;
  const int wave = threadIdx.x / kWave;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int j = 0; j < NS; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i)
        for (int o = a.lanes; o < kWave; o <<= 1) sums[t][j][i] += __shfl_xor(sums[t][j][i], o, kWave);
    __syncthreads();  // the coefficients, and the last table's sums, have been read
    for (int w = 0; w < kWaves; ++w) {
      if (wave == w && in_wave < a.lanes) {
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          const int unit = lane + j * a.lanes;
          if (unit < a.units) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              A* to = shared + unit * V + i;
              *to = w == 0 ? sums[t][j][i] : *to + sums[t][j][i];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int k = threadIdx.x; k < width; k += kThreads)
      a.partial[((int64_t)blockIdx.x * 4 + t) * width + k] = shared[k];
  }
}

// The parameters' gradients from the workgroups' sums: kRnCols copies a workgroup, kParts threads a copy, each over
// every kParts-th row in order, then over the threads in a fixed order.
constexpr int kRnCols = 4;
template <typename X, typename U, bool kCopies>
__global__ __launch_bounds__(kRnThreads) void residual_norm_reduce_kernel(RnArgs<X, U> a, int64_t blocks) {
  using A = typename RnAcc<X>::type;
  constexpr int V = RnUnit<X, U, kCopies>::V, kParts = kRnThreads / kRnCols;
  __shared__ A part[4][kRnWaves][kRnCols];
  const int col = threadIdx.x % kRnCols, from = threadIdx.x / kRnCols;
  const int c = blockIdx.x * kRnCols + col, width = a.units * V;
  const bool live = c < a.copies, scalar = c < a.a0;
  // where the sums hold the copy's first number
  const int at = kCopies ? 2 * c : (scalar ? c : 2 * c - a.a0);
  A s[4] = {A(0), A(0), A(0), A(0)};
  if (live) {
#pragma unroll 4
    for (int64_t b = from; b < blocks; b += kParts)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const A* row = a.partial + (b * 4 + t) * width + at;
        s[t] += scalar ? row[0] : row[0] + row[1];
      }
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    for (int o = kRnCols; o < kWave; o <<= 1) s[t] += __shfl_xor(s[t], o, kWave);
    if (threadIdx.x % kWave < kRnCols) part[t][threadIdx.x / kWave][col] = s[t];
  }
  __syncthreads();
  if (from != 0 || !live) return;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    s[t] = A(0);
#pragma unroll
    for (int w = 0; w < kRnWaves; ++w) s[t] += part[t][w][col];
  }
  const RnPlace p = place_of(a, scalar ? c : 2 * c - a.a0);
  const A scale = a.scaled ? a.scale[p.slot][p.copy] : A(1), gain = a.normalise ? a.gain[p.slot][p.copy] : A(1);
  const A offset = a.offset && scalar ? a.offset[c] : A(0);
  const int C = a.copies;
  A* out = a.dparams;
  out[c] = scale * s[0];
  if (scalar) out[C + c] = scale * s[1];
  out[C + a.a0 + c] = gain * s[0] + offset * s[1];
  out[2 * C + a.a0 + c] = s[2];
  if (scalar) out[3 * C + a.a0 + c] = s[3];
}

// ------------------------------------------------------------------ launch

// Units a lane holds at most, the rows' numbers being registers: 20 numbers of float and bfloat16 rows in the forward,
// 16 in the backward, whose lanes are more (dispatch_rn) and whose sums take as many registers again as its rows; 16 of
// double rows, and of a wide row's copies 32.
template <typename X, bool kCopies, bool kBackward>
constexpr int kMaxUnits = kCopies ? 16 : (sizeof(X) == 8 ? 8 : (kBackward ? 4 : 5));

template <typename X, typename U, bool kCopies, int NS, bool kBackward>
int launch_rn(const RnArgs<X, U>& a, hipStream_t stream, int64_t& blocks) {
  using A = typename RnAcc<X>::type;
  constexpr int kBlock = kBackward ? kRnBackThreads<X, kCopies, NS> : kRnThreads;
  const int64_t rows_per_block = (int64_t)(kBlock / kWave) * (kWave >> a.shift);
  const int width = a.units * RnUnit<X, U, kCopies>::V;
  const size_t lds = sizeof(A) * std::max<size_t>((size_t)kTables * a.D, kBackward ? width : 0);
  const int64_t want = (a.n_rows + rows_per_block - 1) / rows_per_block;
  if constexpr (kBackward) {
    // a row of sums a workgroup: as many as the caller's array was sized for, eight waves a CU
    blocks = std::min<int64_t>(want, std::min<int64_t>(blocks, kBlock == 512 ? 256 : 512));
    hipLaunchKernelGGL((residual_norm_backward_kernel<X, U, kCopies, NS>), dim3((unsigned)blocks), dim3(kBlock), lds,
                       stream, a);
  } else {
    const int64_t slots = resident_blocks(
        reinterpret_cast<const void*>(&residual_norm_forward_kernel<X, U, kCopies, NS>), kBlock, lds);
    blocks = std::min<int64_t>(want, slots > 0 ? slots : 1024);
    hipLaunchKernelGGL((residual_norm_forward_kernel<X, U, kCopies, NS>), dim3((unsigned)blocks), dim3(kBlock), lds,
                       stream, a);
  }
  return check_launch(kBackward ? "residual_norm_backward" : "residual_norm_forward");
}

template <bool kCopies, bool kBackward, typename X, typename U>
int dispatch_rn(RnArgs<X, U>& a, hipStream_t stream, int64_t& blocks) {
  a.units = kCopies ? a.copies : a.D / RnUnit<X, U, kCopies>::V;
  a.scalar_units = kCopies ? a.a0 : a.a0 / RnUnit<X, U, kCopies>::V;
  a.lanes = 1;
  a.shift = 0;
  constexpr int kMost = kMaxUnits<X, kCopies, kBackward>;
  // as few lanes a row as hold it within kMost a lane, or four copies (whose loads are a number each); the backward
  // within three units, since its sums take as many registers again as its rows (float rows of five units a lane: 266
  // registers and one wave a SIMD, of three 180 and two); the widest rows take the whole wave
  constexpr int kLane = kCopies ? 4 : (kBackward ? 3 : (kMost < 5 ? kMost : 5));
  while (a.lanes < kWave && (a.units + a.lanes - 1) / a.lanes > kLane) {
    a.lanes *= 2;
    ++a.shift;
  }
  const int ns = (a.units + a.lanes - 1) / a.lanes;
#define GM_RN_CASE(n)                                                                        \
  if constexpr (n <= kMost) {                                                                \
    if (ns <= n) return launch_rn<X, U, kCopies, n, kBackward>(a, stream, blocks);           \
  }
  GM_RN_CASE(1)
  GM_RN_CASE(2)
  GM_RN_CASE(3)
  GM_RN_CASE(4)
  if constexpr (!kCopies && sizeof(X) != 8) {
    GM_RN_CASE(5)
  } else {
    GM_RN_CASE(8)
    GM_RN_CASE(16)
  }
#undef GM_RN_CASE
  return fail(GM_ERR_UNSUPPORTED, "residual_norm: the row is wider than 1024");
}

template <typename X, typename U>
int fill_rn(RnArgs<X, U>& a, int64_t n_rows, int64_t D, int64_t a0, int64_t nf, const int64_t* offsets,
            const int64_t* mults, double factor, double eps, double next_eps) {
  using A = typename RnAcc<X>::type;
  GM_REQUIRE(n_rows >= 0, "the number of rows must be non-negative");
  GM_REQUIRE(D >= 1 && D <= kRnMaxWidth, "the flat width must lie in 1..1024");
  GM_REQUIRE(nf >= 0 && nf <= kRnMaxFreq, "at most 8 nonzero frequencies");
  GM_REQUIRE(a0 >= 0 && a0 <= D, "a0 must lie in 0..D");
  GM_REQUIRE(nf == 0 || (offsets && mults), "offsets and multiplicities (host arrays) are required");
  GM_REQUIRE(eps > 0 && next_eps > 0, "eps must be positive");
  int64_t next = a0, copies = a0;
  for (int64_t f = 0; f < nf; ++f) {
    GM_REQUIRE(mults[f] >= 1 && offsets[f] == next, "frequency blocks must follow frequency 0 contiguously");
    a.off[f] = (int)offsets[f];
    a.mult[f] = (int)mults[f];
    next += 2 * mults[f];
    copies += mults[f];
  }
  GM_REQUIRE(next == D, "the frequency blocks must fill the flat width");
  a.n_rows = n_rows;
  a.D = (int)D;
  a.a0 = (int)a0;
  a.nf = (int)nf;
  a.copies = (int)copies;
  a.present = (int)nf + (a0 > 0 ? 1 : 0);
  a.factor = (A)factor;
  a.eps = (A)eps;
  a.next_eps = (A)next_eps;
  return GM_OK;
}

// Whole units: frequency 0's and the row's numbers are units, the gates' rows halves of them, and the pointers are
// aligned to them.
template <typename X, typename U>
bool whole_units(const RnArgs<X, U>& a) {
  constexpr int V = RnUnit<X, U, false>::V;
  constexpr size_t ax = V * sizeof(X), au = std::min<size_t>(16, V * sizeof(U));
  if (a.D % V != 0 || a.a0 % V != 0) return false;
  if (a.z && (a.copies % (V / 2) != 0 || !aligned(a.z, ax) || !aligned(a.dz, ax))) return false;
  return aligned(a.x, ax) && aligned(a.u, au) && aligned(a.y, ax) && aligned(a.normed, ax) && aligned(a.dy, ax) &&
         aligned(a.dn, ax) && aligned(a.dx, ax) && aligned(a.du, au);
}

// The parameters' pointers (HOST array, 3 (nf + 1) + 2): the gains by frequency (slot 0 frequency 0), the scales, the
// next gains, then the offsets.  A whole group is given or missing; a slot without copies is not read.
template <typename X, typename U>
int take_parameters(RnArgs<X, U>& a, const void* const* params) {
  using A = typename RnAcc<X>::type;
  GM_REQUIRE(params, "the parameters' pointers (a host array) are required");
  const int slots = a.nf + 1;
  for (int g = 0; g < 3; ++g) {
    const A** to = g == 0 ? a.gain : (g == 1 ? a.scale : a.next_gain);
    int given = 0, wanted = 0;
    for (int f = 0; f < slots; ++f) {
      to[f] = static_cast<const A*>(params[g * slots + f]);
      if (f > 0 || a.a0 > 0) {
        ++wanted;
        given += to[f] != nullptr;
      }
    }
    GM_REQUIRE(given == 0 || given == wanted, "a group of parameters needs a vector of every frequency");
    (g == 0 ? a.normalise : (g == 1 ? a.scaled : a.next)) = given > 0;
  }
  a.offset = a.normalise ? static_cast<const A*>(params[3 * slots]) : nullptr;
  a.next_offset = a.next ? static_cast<const A*>(params[3 * slots + 1]) : nullptr;
  return GM_OK;
}

constexpr int64_t kRnMaxBlocks = 512;  // two of four waves a CU: what the backward's registers leave room for

int64_t rn_blocks(int64_t n_rows) {
  // at least 32 rows a workgroup, so that few rows do not leave many rows of sums to add
  return std::max<int64_t>(1, std::min<int64_t>((n_rows + 31) / 32, kRnMaxBlocks));
}

template <typename X, typename U>
int residual_forward(const X* x, const U* u, const X* z, const void* const* params, int64_t n_rows, int64_t D,
                     int64_t a0, int64_t nf, const int64_t* offsets, const int64_t* mults, double factor, double eps,
                     double next_eps, X* y, X* normed, typename RnAcc<X>::type* stats, void* stream) {
  RnArgs<X, U> a{};
  int rc = fill_rn(a, n_rows, D, a0, nf, offsets, mults, factor, eps, next_eps);
  if (rc == GM_OK) rc = take_parameters(a, params);
  if (rc != GM_OK) return rc;
  if (n_rows == 0) return GM_OK;
  GM_REQUIRE(x && u && y, "x, u and y must be device pointers");
  GM_REQUIRE(!a.next || normed, "normed must be a device pointer where there is a next norm");
  a.x = x;
  a.u = u;
  a.z = z;
  a.y = y;
  a.normed = normed;
  a.stats = stats;
  int64_t blocks = 0;
  return whole_units(a) ? dispatch_rn<false, false>(a, (hipStream_t)stream, blocks)
                        : dispatch_rn<true, false>(a, (hipStream_t)stream, blocks);
}

template <typename X, typename U>
int residual_backward(const X* dy, const X* dn, const X* x, const U* u, const X* z, const void* const* params,
                      const typename RnAcc<X>::type* stats, int64_t n_rows, int64_t D, int64_t a0, int64_t nf,
                      const int64_t* offsets, const int64_t* mults, double factor, X* dx, U* du, X* dz,
                      typename RnAcc<X>::type* partial, typename RnAcc<X>::type* dparams, void* stream) {
  RnArgs<X, U> a{};
  int rc = fill_rn(a, n_rows, D, a0, nf, offsets, mults, factor, 1.0, 1.0);
  if (rc == GM_OK) rc = take_parameters(a, params);
  if (rc != GM_OK) return rc;
  GM_REQUIRE(partial && dparams, "partial and dparams must be device pointers");
  if (n_rows > 0) {
    GM_REQUIRE(x && u && stats && dx && du, "x, u, stats, dx and du must be device pointers");
    GM_REQUIRE(!z || dz, "dz must be a device pointer where there are gates");
    GM_REQUIRE(!dn || a.next, "a gradient of the next norm needs its gains");
  }
  a.dy = dy;
  a.dn = dn;
  a.x = x;
  a.u = u;
  a.z = z;
  a.stats = const_cast<typename RnAcc<X>::type*>(stats);  // read only here
  a.dx = dx;
  a.du = du;
  a.dz = dz;
  a.partial = partial;
  a.dparams = dparams;
  int64_t blocks = n_rows > 0 ? rn_blocks(n_rows) : 0;
  const bool units = whole_units(a);
  const hipStream_t s = (hipStream_t)stream;
  if (n_rows > 0) {
    const int status =
        units ? dispatch_rn<false, true>(a, s, blocks) : dispatch_rn<true, true>(a, s, blocks);
    if (status != GM_OK) return status;
  }
  const dim3 grid((unsigned)((a.copies + kRnCols - 1) / kRnCols));
  if (units)
    hipLaunchKernelGGL((residual_norm_reduce_kernel<X, U, false>), grid, dim3(kRnThreads), 0, s, a, blocks);
  else
    hipLaunchKernelGGL((residual_norm_reduce_kernel<X, U, true>), grid, dim3(kRnThreads), 0, s, a, blocks);
  return check_launch("residual_norm_backward (reduce)");
}

}  // namespace
}  // namespace gm

extern "C" int64_t gm_residual_norm_partial_rows(int64_t n_rows) { return n_rows > 0 ? 4 * gm::rn_blocks(n_rows) : 4; }

// X, U: the rows' and the branch's element types in the C signature, TX, TU the kernels'; A the parameters'.
#define GM_RESIDUAL_ENTRY(SFX, X, U, TX, TU, A)                                                                       \
  extern "C" int gm_residual_norm_forward_##SFX(const X* x, const U* u, const X* z, const void* const* params,        \
                                                int64_t n_rows, int64_t D, int64_t a0, int64_t nf,                    \
                                                const int64_t* offsets, const int64_t* mults, double factor,          \
                                                double eps, double next_eps, X* y, X* normed, A* stats,               \
                                                void* stream) {                                                       \
    return gm::residual_forward<TX, TU>(reinterpret_cast<const TX*>(x), reinterpret_cast<const TU*>(u),               \
                                        reinterpret_cast<const TX*>(z), params, n_rows, D, a0, nf, offsets, mults,    \
                                        factor, eps, next_eps, reinterpret_cast<TX*>(y),                              \
                                        reinterpret_cast<TX*>(normed), stats, stream);                                \
  }                                                                                                                   \
  extern "C" int gm_residual_norm_backward_##SFX(                                                                     \
      const X* dy, const X* dn, const X* x, const U* u, const X* z, const void* const* params, const A* stats,        \
      int64_t n_rows, int64_t D, int64_t a0, int64_t nf, const int64_t* offsets, const int64_t* mults, double factor, \
      X* dx, U* du, X* dz, A* partial, A* dparams, void* stream) {                                                    \
    return gm::residual_backward<TX, TU>(reinterpret_cast<const TX*>(dy), reinterpret_cast<const TX*>(dn),            \
                                         reinterpret_cast<const TX*>(x), reinterpret_cast<const TU*>(u),              \
                                         reinterpret_cast<const TX*>(z), params, stats, n_rows, D, a0, nf, offsets,   \
                                         mults, factor, reinterpret_cast<TX*>(dx), reinterpret_cast<TU*>(du),         \
                                         reinterpret_cast<TX*>(dz), partial, dparams, stream);                        \
  }

GM_RESIDUAL_ENTRY(f32, float, float, float, float, float)
GM_RESIDUAL_ENTRY(f64, double, double, double, double, double)
GM_RESIDUAL_ENTRY(bf16, uint16_t, uint16_t, gm::rbf16, gm::rbf16, float)
GM_RESIDUAL_ENTRY(bf16_f32, uint16_t, float, gm::rbf16, float, float)
