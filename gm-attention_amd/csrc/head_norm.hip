// The norm and rotation of rows of heads, of one or two sets of rows (queries and
// keys) over the same nodes.  For every head's numbers x (P of them) of a node i:
//   xhat = x / sqrt(mean x^2 + eps)
//   y    = exp(i theta(i, slot)) (gain xhat),  theta = sum_a position(i, a) frequency(a, slot)
// a gain a copy, the same for every head, and a slot a complex copy; copies of
// frequency 0 turn in pairs (2 j, 2 j + 1), a last odd one stays.  Norm, gains and
// angles may each be left out.  Backward, with d = exp(-i theta) dy and t = gain d:
//   dgain = sum over nodes and heads of d xhat
//   dx    = (t - xhat mean(t xhat)) / sqrt(mean x^2 + eps)
//
// A pass reads its rows once and writes once, and the bytes bound it: 524,288 rows of 160 of queries and keys each take
// 258 us forward and 420 backward in float (5.2 and 4.8 TB/s), 126 and 230 in bfloat16 (5.3 and 4.4: its registers
// leave two waves a SIMD).  Angles are made in the pass, in double up to the whole turns (a far position's angle has no
// bits left in float), once for all heads and both sets; sums of a head are in double from what a lane (a unit) adds in
// float, so that no row overflows.
//
// The lane kernels hold a unit of a head a lane and need no other wave's numbers.  Layouts without such units (odd
// copies, frequencies above 2, rows at odd addresses) and double take the general kernels, where a thread holds the
// same piece of a row for all the rows of its workgroup and a head's squares meet in LDS between barriers (305 and
// 497 us for the float rows above, 245 and 507 for the bfloat16 ones).  All are persistent; gains, and sums for their
// gradients, stay in registers over a workgroup's rows, whose sums are added in a fixed order, no atomics.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "edge_units.hpp"
#include "heads.hpp"
#include "partial_sum.hpp"

namespace gm {
namespace {

constexpr int kHnMaxHeads = 64;
constexpr int kHnMaxAxes = 8;
constexpr int kHnThreads = 576;       // at most: a row of 1,024 numbers has up to 544 units of two
constexpr int kHnPartialRows = 2048;  // workgroups of the backward, at most

template <typename T, typename R>
struct HnArgs {
  HeadsLayout L;
  int copies, slots, numbers;     // a head's copies, angles, numbers
  int units, groups, parts;       // a row's units; rows a workgroup takes at once; lanes that add a head's squares
  int axes;                       // 0: no rotation
  bool normalise;
  int64_t n_rows;
  const R* x[2];
  int64_t stride[2];
  const T* gain[2];               // (copies) or null
  R* y[2];                        // (n_rows, D)
  const R* dy[2];                 // (n_rows, D)
  R* dx[2];                       // (n_rows, D)
  T* partial;                     // (workgroups, sets, copies) or null
  const double* positions;        // (n_rows, axes)
  const double* frequencies;      // (axes, slots)
  double eps, share;              // share: 1 / numbers
};

// Unit u of a row: `width` numbers from column `col` (V but for a last odd scalar), the copy of each among its head's,
// the first pair's slot (-1: no pair).
template <int V>
struct HnUnit {
  int col, width, head, slot;
  int copy[V];
};

// Units a head at a frequency.
template <int V>
__host__ __device__ __forceinline__ int hn_units(int n, int a) {
  return n == 0 ? (a + V - 1) / V : a / (V / 2);
}

template <int V>
__device__ HnUnit<V> hn_unit(const HeadsLayout& L, int u) {
  HnUnit<V> r{};
  int copies = 0, slots = 0;
  for (int f = 0; f < L.F; ++f) {
    const int n = L.n[f], a = L.a[f], per = hn_units<V>(n, a);
    if (u >= 0 && u < L.H * per) {
      const int i = u % per, first = n == 0 ? V * i : V / 2 * i;
      r.head = u / per;
      r.col = L.off[f] + (n == 0 ? r.head * a + first : 2 * (r.head * a + first));
      r.width = n == 0 && a - first < V ? a - first : V;
      r.slot = r.width < 2 ? -1 : slots + (n == 0 ? first / 2 : first);
#pragma unroll
      for (int j = 0; j < V; ++j) r.copy[j] = copies + first + (n == 0 ? (j < r.width ? j : 0) : j / 2);
      return r;
    }
    u -= L.H * per;
    copies += a;
    slots += n == 0 ? a / 2 : a;
  }
  return r;
}

template <int V, typename T, typename R>
__device__ __forceinline__ void hn_load(const R* p, int width, T (&v)[V]) {
  if constexpr (V == 4 && !std::is_same<T, double>::value) {
    load_w<4>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < width ? row_widen(p[j]) : T(0);
  }
}
template <int V, typename T, typename R>
__device__ __forceinline__ void hn_store(R* p, int width, const T (&v)[V]) {
  if constexpr (V == 4 && !std::is_same<T, double>::value) {
    store_w<4>(p, v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < width) row_narrow(v[j], p[j]);
  }
}

__device__ __forceinline__ void hn_sincos(double turns, float& s, float& c) { sincospif(2.f * (float)turns, &s, &c); }
__device__ __forceinline__ void hn_sincos(double turns, double& s, double& c) { sincospi(2.0 * turns, &s, &c); }

// (cos, sin) of a row's angle in a slot.
template <typename T, typename R>
__device__ __forceinline__ void hn_angle(const HnArgs<T, R>& a, int64_t row, int slot, T& c, T& s) {
  double theta = 0.0;
  for (int axis = 0; axis < a.axes; ++axis)
    theta = fma(a.positions[row * a.axes + axis], a.frequencies[axis * a.slots + slot], theta);
  const double turns = theta * 0.15915494309189535;
  hn_sincos(turns - rint(turns), s, c);
}

// (cos, sin) of the angles of `rows` rows from `first`, into LDS.
template <typename T, typename R>
__device__ __forceinline__ void hn_angles(const HnArgs<T, R>& a, int64_t first, int rows, T* cs) {
  for (int i = threadIdx.x; i < rows * a.slots; i += blockDim.x) {
    const int k = i / a.slots, slot = i - k * a.slots;
    const int64_t row = first + k < a.n_rows ? first + k : a.n_rows - 1;
    hn_angle(a, row, slot, cs[2 * i], cs[2 * i + 1]);
  }
}

// The pairs of a unit turned by their slots' angles, `back` against them.
template <int V, typename T>
__device__ __forceinline__ void hn_turn(T (&v)[V], const T* cs, bool back) {
#pragma unroll
  for (int j = 0; j < V; j += 2) {
    const T c = cs[j], s = back ? -cs[j + 1] : cs[j + 1];
    const T v0 = v[j], v1 = v[j + 1];
    v[j] = c * v0 - s * v1;
    v[j + 1] = c * v1 + s * v0;
  }
}

// 1 / sqrt, for float to better than its half step: the approximation in double and a Newton step (of zero and
// infinity the approximation).
template <typename T>
__device__ __forceinline__ double hn_rsqrt(double v) {
  if constexpr (sizeof(T) == 8) return 1.0 / sqrt(v);
  const double y = __builtin_amdgcn_rsq(v);
  const double refined = y * fma(-0.5 * v * y, y, 1.5);
  return v > 0.0 && v < (double)INFINITY ? refined : y;
}
// Sum of a_j b_j in float (two sums, of even and odd j); where that is out of float's range, or near zero (small terms,
// or large ones that cancel), once more in double.
template <int V>
__device__ __forceinline__ double hn_dot(const float (&a)[V], const float (&b)[V]) {
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int j = 0; j + 1 < V; j += 2) {
    s = fmaf(a[j], b[j], s);
    t = fmaf(a[j + 1], b[j + 1], t);
  }
  if constexpr (V % 2) s = fmaf(a[V - 1], b[V - 1], s);
  s += t;
  if (fabsf(s) > 1e-30f && fabsf(s) < INFINITY) return (double)s;
  double wide = 0.0;
#pragma unroll
  for (int j = 0; j < V; ++j) wide = fma((double)a[j], (double)b[j], wide);
  return wide;
}
template <int V>
__device__ __forceinline__ double hn_dot(const double (&a)[V], const double (&b)[V]) {
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < V; ++j) s = fma(a[j], b[j], s);
  return s;
}

// Sum over a head's units of sums[..] (one row's units), shared by `parts` lanes; all of them get it.
template <int V, typename T, typename R>
__device__ __forceinline__ double hn_head_sum(const HnArgs<T, R>& a, const double* sums, int head, int part) {
  double s = 0.0;
  int base = 0;
  for (int f = 0; f < a.L.F; ++f) {
    const int per = hn_units<V>(a.L.n[f], a.L.a[f]);
    for (int i = part; i < per; i += a.parts) s += sums[base + head * per + i];
    base += a.L.H * per;
  }
  for (int o = 1; o < a.parts; o <<= 1) s += __shfl_xor(s, o, kWave);
  return s;
}

// LDS: the squares (and, backward, the products) of the workgroup's rows, the heads' 1 / sqrt (and means), the angles.
template <typename T>
struct HnLds {
  double* sums;  // (kinds, sets, rows, units)
  T* heads;      // (kinds, sets, rows, H)
  T* cs;         // (rows, slots, 2)
};
template <typename T, typename R>
__host__ __device__ inline size_t hn_lds(const HnArgs<T, R>& a, int kinds, int sets, int rows, size_t& heads,
                                         size_t& cs) {
  heads = a.normalise ? (size_t)kinds * sets * rows * a.units * sizeof(double) : 0;
  cs = heads + (a.normalise ? ((size_t)kinds * sets * rows * a.L.H * sizeof(T) + 15) / 16 * 16 : 0);
  return cs + (a.axes ? (size_t)rows * a.slots * 2 * sizeof(T) : 0);
}

template <typename T, typename R, int V, int NS, int TR>
__global__ __launch_bounds__(kHnThreads) void head_norm_forward(HnArgs<T, R> a) {
  extern __shared__ __align__(16) char hn_mem[];
  const int rows = a.groups * TR, u = threadIdx.x % a.units, group = threadIdx.x / a.units;
  const bool live = group < a.groups;
  size_t heads_at, cs_at;
  hn_lds(a, 1, NS, rows, heads_at, cs_at);
  double* sums = reinterpret_cast<double*>(hn_mem);
  T* heads = reinterpret_cast<T*>(hn_mem + heads_at);
  T* cs = reinterpret_cast<T*>(hn_mem + cs_at);
  const HnUnit<V> unit = hn_unit<V>(a.L, u);
  T gain[NS][V];
#pragma unroll
  for (int st = 0; st < NS; ++st)
#pragma unroll
    for (int j = 0; j < V; ++j) gain[st][j] = a.gain[st] ? a.gain[st][unit.copy[j]] : T(1);
  const int64_t tiles = (a.n_rows + rows - 1) / rows;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t first = tile * rows;
    T v[NS][TR][V];
    if (live) {
#pragma unroll
      for (int st = 0; st < NS; ++st)
#pragma unroll
        for (int k = 0; k < TR; ++k) {
          const int64_t row = first + k * a.groups + group;
          hn_load<V>(a.x[st] + (row < a.n_rows ? row : a.n_rows - 1) * a.stride[st] + unit.col, unit.width, v[st][k]);
        }
    }
    __syncthreads();  // the tile before has read its angles and norms
    if (a.axes) hn_angles(a, first, rows, cs);
    if (a.normalise) {
      if (live) {
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
          for (int k = 0; k < TR; ++k) {
            sums[(st * rows + k * a.groups + group) * a.units + u] = hn_dot<V>(v[st][k], v[st][k]);
          }
      }
      __syncthreads();
      const int tasks = NS * rows * a.L.H, part = threadIdx.x % a.parts;
      for (int t = threadIdx.x / a.parts; t < tasks; t += blockDim.x / a.parts) {
        const double s = hn_head_sum<V>(a, sums + t / a.L.H * a.units, t % a.L.H, part);
        if (part == 0) heads[t] = (T)hn_rsqrt<T>(fma(s, a.share, a.eps));
      }
    }
    __syncthreads();
    if (live) {
#pragma unroll
      for (int k = 0; k < TR; ++k) {
        const int at = k * a.groups + group;
        const int64_t row = first + at;
        if (row >= a.n_rows) break;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          const T inv = a.normalise ? heads[(st * rows + at) * a.L.H + unit.head] : T(1);
          T y[V];
#pragma unroll
          for (int j = 0; j < V; ++j) y[j] = gain[st][j] * (v[st][k][j] * inv);
          if (a.axes && unit.slot >= 0) hn_turn<V>(y, cs + 2 * (at * a.slots + unit.slot), false);
          hn_store<V>(a.y[st] + row * a.L.D + unit.col, unit.width, y);
        }
      }
    }
  }
}

template <typename T, typename R, int V, int NS, int TR>
__global__ __launch_bounds__(kHnThreads) void head_norm_backward(HnArgs<T, R> a) {
  extern __shared__ __align__(16) char hn_mem[];
  const int rows = a.groups * TR, u = threadIdx.x % a.units, group = threadIdx.x / a.units;
  const bool live = group < a.groups;
  size_t heads_at, cs_at;
  hn_lds(a, 2, NS, rows, heads_at, cs_at);
  double* sums = reinterpret_cast<double*>(hn_mem);
  T* heads = reinterpret_cast<T*>(hn_mem + heads_at);
  T* cs = reinterpret_cast<T*>(hn_mem + cs_at);
  const int products = NS * rows * a.units, means = NS * rows * a.L.H;
  const HnUnit<V> unit = hn_unit<V>(a.L, u);
  T gain[NS][V], acc[NS][V];
#pragma unroll
  for (int st = 0; st < NS; ++st)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      gain[st][j] = a.gain[st] ? a.gain[st][unit.copy[j]] : T(1);
      acc[st][j] = T(0);
    }
  const int64_t tiles = (a.n_rows + rows - 1) / rows;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t first = tile * rows;
    T v[NS][TR][V], d[NS][TR][V];
    if (live) {
#pragma unroll
      for (int st = 0; st < NS; ++st)
#pragma unroll
        for (int k = 0; k < TR; ++k) {
          const int64_t row = first + k * a.groups + group, at = row < a.n_rows ? row : a.n_rows - 1;
          hn_load<V>(a.x[st] + at * a.stride[st] + unit.col, unit.width, v[st][k]);
          hn_load<V>(a.dy[st] + at * a.L.D + unit.col, unit.width, d[st][k]);
        }
    }
    __syncthreads();  // the tile before has read its angles and means
    if (a.axes) {
      hn_angles(a, first, rows, cs);
      __syncthreads();
      if (live && unit.slot >= 0) {
#pragma unroll
        for (int k = 0; k < TR; ++k) {
          const T* turn = cs + 2 * ((k * a.groups + group) * a.slots + unit.slot);
#pragma unroll
          for (int st = 0; st < NS; ++st) hn_turn<V>(d[st][k], turn, true);
        }
      }
    }
    if (a.normalise) {
      if (live) {
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
          for (int k = 0; k < TR; ++k) {
            T t[V];
#pragma unroll
            for (int j = 0; j < V; ++j) t[j] = gain[st][j] * d[st][k][j];
            const int at = (st * rows + k * a.groups + group) * a.units + u;
            sums[at] = hn_dot<V>(v[st][k], v[st][k]);
            sums[products + at] = hn_dot<V>(t, v[st][k]);
          }
      }
      __syncthreads();
      const int part = threadIdx.x % a.parts;
      for (int t = threadIdx.x / a.parts; t < means; t += blockDim.x / a.parts) {
        const double* row = sums + t / a.L.H * a.units;
        const double s = hn_head_sum<V>(a, row, t % a.L.H, part);
        const double m = hn_head_sum<V>(a, row + products, t % a.L.H, part);
        if (part == 0) {
          const double inv = hn_rsqrt<T>(fma(s, a.share, a.eps));
          heads[t] = (T)inv;
          heads[means + t] = (T)(m * inv * a.share);
        }
      }
      __syncthreads();
    }
    if (live) {
#pragma unroll
      for (int k = 0; k < TR; ++k) {
        const int at = k * a.groups + group;
        const int64_t row = first + at;
        if (row >= a.n_rows) break;
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          const int h = (st * rows + at) * a.L.H + unit.head;
          const T inv = a.normalise ? heads[h] : T(1), mean = a.normalise ? heads[means + h] : T(0);
          T dx[V];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const T hat = v[st][k][j] * inv;
            acc[st][j] += d[st][k][j] * hat;
            dx[j] = inv * (gain[st][j] * d[st][k][j] - hat * mean);
          }
          hn_store<V>(a.dx[st] + row * a.L.D + unit.col, unit.width, dx);
        }
      }
    }
  }
  if (!a.partial) return;
  // the workgroup's sums: over its groups of rows and the heads, a copy's two numbers together
  T* held = reinterpret_cast<T*>(hn_mem);  // (groups, units, V)
#pragma unroll
  for (int st = 0; st < NS; ++st) {
    __syncthreads();
    if (live) {
#pragma unroll
      for (int j = 0; j < V; ++j) held[(group * a.units + u) * V + j] = acc[st][j];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.copies; c += blockDim.x) {
      int f = 0, local = c, base = 0;
      while (local >= a.L.a[f]) {
        local -= a.L.a[f];
        base += a.L.H * hn_units<V>(a.L.n[f], a.L.a[f]);
        ++f;
      }
      const int n = a.L.n[f], per = hn_units<V>(n, a.L.a[f]), wide = n == 0 ? V : V / 2;
      const int i = local / wide, j = local % wide * (n == 0 ? 1 : 2);
      T s = T(0);
      for (int g = 0; g < a.groups; ++g)
        for (int h = 0; h < a.L.H; ++h) {
          const T* at = held + (g * a.units + base + h * per + i) * V + j;
          s += n == 0 ? at[0] : at[0] + at[1];
        }
      a.partial[((int64_t)blockIdx.x * NS + st) * a.copies + c] = s;
    }
  }
}

// ------------------------------------------------------------- lane kernels
// A head's copies as `per` units of (A0, A1, A2) copies of frequencies 0, 1, 2, a lane a unit: a head's sums are in
// its own lanes, so a wave's rows need nothing of the other waves.  A row's angles are made by its lanes, each some of
// them, and handed over through the wave's LDS.

struct HnShape {
  int a0, a1, a2;
};
struct HnLanes {
  int per, lanes, rows;  // units a head; lanes a row, rows a wave
  int base[3];           // the frequencies' flat offsets
  int c0, c1, c2;        // a head's copies at frequencies 0, 1, 2
};

template <int A0, int A1, int A2>
struct HnRow {
  static constexpr int W0 = A0, W1 = 2 * A1, W2 = 2 * A2, N = W0 + W1 + W2, C = A0 + A1 + A2;
  static constexpr int kPairs = A0 / 2, S = kPairs + A1 + A2;  // pairs of scalars; the unit's slots
  template <typename R>
  static __device__ __forceinline__ void load(const R* row, const HnLanes& w, int u, float (&v)[N]) {
    if constexpr (W0 > 0) load_piece<W0>(row + w.base[0] + u * W0, v);
    if constexpr (W1 > 0) load_piece<W1>(row + w.base[1] + u * W1, v + W0);
    if constexpr (W2 > 0) load_piece<W2>(row + w.base[2] + u * W2, v + W0 + W1);
  }
  template <typename R>
  static __device__ __forceinline__ void store(R* row, const HnLanes& w, int u, const float (&v)[N]) {
    if constexpr (W0 > 0) store_piece<W0>(row + w.base[0] + u * W0, v);
    if constexpr (W1 > 0) store_piece<W1>(row + w.base[1] + u * W1, v + W0);
    if constexpr (W2 > 0) store_piece<W2>(row + w.base[2] + u * W2, v + W0 + W1);
  }
  template <int W, typename R>
  static __device__ __forceinline__ void load_piece(const R* p, float* v) {
    if constexpr (W == 8 && sizeof(R) == 2) {
      const uint4 x = *reinterpret_cast<const uint4*>(p);
      const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(word[i] << 16);
        v[2 * i + 1] = __uint_as_float(word[i] & 0xFFFF0000u);
      }
    } else {
      load_w<W>(p, v);
    }
  }
  template <int W, typename R>
  static __device__ __forceinline__ void store_piece(R* p, const float* v) {
    if constexpr (W == 8 && sizeof(R) == 2)
      *reinterpret_cast<uint4*>(p) = make_uint4(row_pack(v[0], v[1]), row_pack(v[2], v[3]), row_pack(v[4], v[5]),
                                                row_pack(v[6], v[7]));
    else
      store_w<W>(p, v);
  }
  // the copy of a head that the unit's number i belongs to
  static __device__ __forceinline__ int copy(const HnLanes& w, int own, int i) {
    if (i < W0) return own * A0 + i;
    if (i < W0 + W1) return w.c0 + own * A1 + (i - W0) / 2;
    return w.c0 + w.c1 + own * A2 + (i - W0 - W1) / 2;
  }
  // the head's slot of the unit's pair j
  static __device__ __forceinline__ int slot(const HnLanes& w, int own, int j) {
    if (j < kPairs) return own * kPairs + j;
    if (j < kPairs + A1) return w.c0 / 2 + own * A1 + j - kPairs;
    return w.c0 / 2 + w.c1 + own * A2 + j - kPairs - A1;
  }
  static constexpr int pair(int j) { return j < kPairs ? 2 * j : W0 + 2 * (j - kPairs); }
  static __device__ __forceinline__ void turn(float (&v)[N], const float2 (&cs)[S > 0 ? S : 1], bool back) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
      const float c = cs[j].x, s = back ? -cs[j].y : cs[j].y, v0 = v[pair(j)], v1 = v[pair(j) + 1];
      v[pair(j)] = c * v0 - s * v1;
      v[pair(j) + 1] = c * v1 + s * v0;
    }
  }
};

__device__ __forceinline__ double hn_lane_sum(double v, int per) {
  for (int o = 1; o < per; o <<= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// The angles of a lane's pairs; `cs` the wave's LDS (rows, slots).
template <typename U, typename R>
__device__ __forceinline__ void hn_lane_angles(const HnArgs<float, R>& a, const HnLanes& w, int64_t row, int r, int u,
                                               int own, float2* cs, float2 (&out)[U::S > 0 ? U::S : 1]) {
  wave_lds();  // the rows before have been read
  if (r < w.rows)
    for (int slot = u; slot < a.slots; slot += w.lanes)
      hn_angle(a, row, slot, cs[r * a.slots + slot].x, cs[r * a.slots + slot].y);
  wave_lds();
#pragma unroll
  for (int j = 0; j < U::S; ++j) out[j] = cs[(r < w.rows ? r : 0) * a.slots + U::slot(w, own, j)];
}

template <typename R, typename U, int NS>
__global__ __launch_bounds__(256) void head_norm_forward_lanes(HnArgs<float, R> a, HnLanes w) {
  extern __shared__ __align__(16) char hn_mem[];
  const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
  float2* cs = reinterpret_cast<float2*>(hn_mem) + wave * w.rows * a.slots;
  const int r = lane / w.lanes, u = lane % w.lanes, own = u % w.per;
  float gain[NS][U::N];
#pragma unroll
  for (int st = 0; st < NS; ++st)
#pragma unroll
    for (int i = 0; i < U::N; ++i) gain[st][i] = a.gain[st] ? a.gain[st][U::copy(w, own, i)] : 1.f;
  const int64_t step = (int64_t)gridDim.x * kWavesPerBlock * w.rows;
  for (int64_t first = ((int64_t)blockIdx.x * kWavesPerBlock + wave) * w.rows; first < a.n_rows; first += step) {
    const bool live = r < w.rows && first + r < a.n_rows;
    const int64_t row = live ? first + r : first;
    float v[NS][U::N];
#pragma unroll
    for (int st = 0; st < NS; ++st) U::load(a.x[st] + row * a.stride[st], w, u, v[st]);
    float2 turn[U::S > 0 ? U::S : 1];
    if (a.axes) hn_lane_angles<U>(a, w, row, r, u, own, cs, turn);
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      const double square = hn_lane_sum(hn_dot(v[st], v[st]), w.per);
      const float inv = a.normalise ? (float)hn_rsqrt<float>(fma(square, a.share, a.eps)) : 1.f;
#pragma unroll
      for (int i = 0; i < U::N; ++i) v[st][i] = gain[st][i] * (v[st][i] * inv);
      if (a.axes) U::turn(v[st], turn, false);
      if (live) U::store(a.y[st] + row * a.L.D, w, u, v[st]);
    }
  }
}

template <typename R, typename U, int NS>
__global__ __launch_bounds__(256) void head_norm_backward_lanes(HnArgs<float, R> a, HnLanes w) {
  extern __shared__ __align__(16) char hn_mem[];
  const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
  float2* cs = reinterpret_cast<float2*>(hn_mem) + wave * w.rows * a.slots;
  const int r = lane / w.lanes, u = lane % w.lanes, own = u % w.per;
  float gain[NS][U::N], acc[NS][U::C];
#pragma unroll
  for (int st = 0; st < NS; ++st) {
#pragma unroll
    for (int i = 0; i < U::N; ++i) gain[st][i] = a.gain[st] ? a.gain[st][U::copy(w, own, i)] : 1.f;
#pragma unroll
    for (int c = 0; c < U::C; ++c) acc[st][c] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * kWavesPerBlock * w.rows;
  for (int64_t first = ((int64_t)blockIdx.x * kWavesPerBlock + wave) * w.rows; first < a.n_rows; first += step) {
    const bool live = r < w.rows && first + r < a.n_rows;
    const int64_t row = live ? first + r : first;
    float v[NS][U::N], d[NS][U::N];
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      U::load(a.x[st] + row * a.stride[st], w, u, v[st]);
      U::load(a.dy[st] + row * a.L.D, w, u, d[st]);
    }
    float2 turn[U::S > 0 ? U::S : 1];
    if (a.axes) hn_lane_angles<U>(a, w, row, r, u, own, cs, turn);
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      if (a.axes) U::turn(d[st], turn, true);
      float t[U::N], inv = 1.f, mean = 0.f;
#pragma unroll
      for (int i = 0; i < U::N; ++i) t[i] = gain[st][i] * d[st][i];
      if (a.normalise) {
        const double wide = hn_rsqrt<float>(fma(hn_lane_sum(hn_dot(v[st], v[st]), w.per), a.share, a.eps));
        inv = (float)wide;
        mean = (float)(hn_lane_sum(hn_dot(t, v[st]), w.per) * wide * a.share);
      }
#pragma unroll
      for (int i = 0; i < U::N; ++i) {
        const float hat = v[st][i] * inv;
        const int c = i < U::W0 ? i : U::W0 + (i - U::W0) / 2;
        acc[st][c] = fmaf(live ? d[st][i] : 0.f, hat, acc[st][c]);
        t[i] = inv * (t[i] - hat * mean);
      }
      if (live) U::store(a.dx[st] + row * a.L.D, w, u, t);
    }
  }
  if (!a.partial) return;
  // the workgroup's sums, in the order of its waves, rows and heads
  float* held = reinterpret_cast<float*>(hn_mem);  // (C, 256)
#pragma unroll
  for (int st = 0; st < NS; ++st) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < U::C; ++c) held[c * 256 + threadIdx.x] = acc[st][c];
    __syncthreads();
    for (int c = threadIdx.x; c < a.copies; c += blockDim.x) {
      const int freq = c < w.c0 ? 0 : (c < w.c0 + w.c1 ? 1 : 2);
      const int wide = freq == 0 ? U::W0 : (freq == 1 ? U::W1 / 2 : U::W2 / 2);
      const int local = c - (freq == 0 ? 0 : (freq == 1 ? w.c0 : w.c0 + w.c1)), unit = local / wide;
      const int at = local % wide + (freq == 0 ? 0 : (freq == 1 ? U::W0 : U::W0 + U::W1 / 2));
      float s = 0.f;
      for (int wv = 0; wv < kWavesPerBlock; ++wv)
        for (int row = 0; row < w.rows; ++row)
          for (int h = unit; h < w.lanes; h += w.per) s += held[at * 256 + wv * kWave + row * w.lanes + h];
      a.partial[((int64_t)blockIdx.x * NS + st) * a.copies + c] = s;
    }
  }
}

// ------------------------------------------------------------------- launch

// Whether units of four numbers serve: whole units of one frequency in every head, and rows at whole units.
template <typename T, typename R>
bool hn_wide(const HnArgs<T, R>& a, int sets, bool backward) {
  if (sizeof(T) == 8) return false;
  for (int f = 0; f < a.L.F; ++f)
    if (a.L.a[f] % (a.L.n[f] == 0 ? 4 : 2) != 0 || a.L.off[f] % 4 != 0) return false;
  const size_t unit = 4 * sizeof(R);
  if (a.L.D % 4 != 0) return false;
  for (int st = 0; st < sets; ++st) {
    if (a.stride[st] % 4 != 0 || !aligned(a.x[st], unit)) return false;
    if (backward ? !(aligned(a.dy[st], unit) && aligned(a.dx[st], unit)) : !aligned(a.y[st], unit)) return false;
  }
  return true;
}

template <typename T, typename R, int V, int NS, bool kBackward>
int hn_launch(HnArgs<T, R> a, T* dgain, hipStream_t stream) {
  constexpr int TR = kBackward ? 2 : 4;
  a.units = 0;
  int head_units = 0;
  for (int f = 0; f < a.L.F; ++f) head_units += hn_units<V>(a.L.n[f], a.L.a[f]);
  a.units = a.L.H * head_units;
  // about 256 threads, whole waves as far as the units allow; no more rows than there are
  int best = 1;
  double fill = 0.0;
  for (int g = 1; g * a.units <= 384; ++g) {
    const int used = g * a.units;
    const double here = (double)used / ((used + 63) / 64 * 64) * (used < 192 ? used / 192.0 : 1.0);
    if (here > fill + 1e-9) {
      fill = here;
      best = g;
    }
    if ((int64_t)g * TR >= a.n_rows) break;
  }
  a.groups = best;
  const int threads = (a.groups * a.units + 63) / 64 * 64;
  const int rows = a.groups * TR;
  for (a.parts = 1; a.parts < 64 && a.parts * 2 <= head_units && NS * rows * a.L.H * a.parts * 2 <= threads;)
    a.parts *= 2;
  size_t unused0, unused1;
  size_t lds = hn_lds(a, kBackward ? 2 : 1, NS, rows, unused0, unused1);
  if (kBackward && a.partial) lds = std::max(lds, (size_t)a.groups * a.units * V * sizeof(T));
  using Kernel = void (*)(HnArgs<T, R>);
  constexpr Kernel kernel =
      kBackward ? &head_norm_backward<T, R, V, NS, TR> : &head_norm_forward<T, R, V, NS, TR>;
  if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess)
    return check_launch("head_norm (LDS)");
  const int64_t tiles = (a.n_rows + rows - 1) / rows;
  const int64_t resident = resident_blocks(reinterpret_cast<const void*>(kernel), threads, lds);
  const int64_t most = std::min<int64_t>(kHnPartialRows, resident > 0 ? resident : kHnPartialRows);
  const int64_t blocks = std::min(tiles, most);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), lds, stream, a);
  if (kBackward && a.partial) launch_partial_sum<T>(a.partial, blocks, NS * a.copies, dgain, stream);
  return check_launch("head_norm");
}

// A workgroup of four waves of whole rows each; resident ones.
template <typename R, int A0, int A1, int A2, int NS, bool kBackward>
int hn_launch_lanes(const HnArgs<float, R>& a, const HnLanes& w, float* dgain, hipStream_t stream) {
  using U = HnRow<A0, A1, A2>;
  using Kernel = void (*)(HnArgs<float, R>, HnLanes);
  constexpr Kernel kernel = kBackward ? &head_norm_backward_lanes<R, U, NS> : &head_norm_forward_lanes<R, U, NS>;
  size_t lds = a.axes ? (size_t)kWavesPerBlock * w.rows * a.slots * sizeof(float2) : 0;
  if (kBackward && a.partial) lds = std::max(lds, (size_t)U::C * 256 * sizeof(float));
  const int64_t per = kWavesPerBlock * w.rows, tiles = (a.n_rows + per - 1) / per;
  const int64_t resident = resident_blocks(reinterpret_cast<const void*>(kernel), 256, lds);
  const int64_t most = std::min<int64_t>(kHnPartialRows, resident > 0 ? resident : kHnPartialRows);
  const int64_t blocks = std::min(tiles, most);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, stream, a, w);
  if (kBackward && a.partial) launch_partial_sum<float>(a.partial, blocks, NS * a.copies, dgain, stream);
  return check_launch("head_norm");
}

// The units of the lane kernels: pieces of 16 bytes at the frequencies above 0 where the copies allow, at frequency 0
// whole pairs of scalars.
constexpr HnShape kHnFloat[] = {{2, 2, 2}, {4, 2, 2}, {4, 2, 0}, {2, 2, 0}, {4, 2, 1}, {4, 0, 0}, {0, 2, 2}, {2, 1, 1}};
constexpr HnShape kHnHalf[] = {{4, 4, 4}, {8, 4, 4}, {4, 4, 0}, {8, 4, 2}, {8, 0, 0}, {0, 4, 4}, {2, 2, 2}, {2, 1, 1}};

// The shape's index, or -1: the layout has other frequencies, no such units, or rows beside their alignment.
template <typename R>
int hn_shape(const HnArgs<float, R>& a, int sets, bool backward, HnLanes& w) {
  int c[3] = {0, 0, 0};
  for (int f = 0; f < 3; ++f) w.base[f] = 0;
  for (int f = 0; f < a.L.F; ++f) {
    if (a.L.n[f] > 2) return -1;
    c[a.L.n[f]] = a.L.a[f];
    w.base[a.L.n[f]] = a.L.off[f];
  }
  w.c0 = c[0];
  w.c1 = c[1];
  w.c2 = c[2];
  constexpr int kCount = 8;
  const HnShape(&shapes)[kCount] = sizeof(R) == 4 ? kHnFloat : kHnHalf;
  for (int i = 0; i < kCount; ++i) {
    const HnShape& s = shapes[i];
    for (w.per = 1; w.per * a.L.H <= kWave; w.per *= 2) {
      if (c[0] != w.per * s.a0 || c[1] != w.per * s.a1 || c[2] != w.per * s.a2) continue;
      const int width[3] = {s.a0, 2 * s.a1, 2 * s.a2};
      size_t unit = 1;
      for (int f = 0; f < 3; ++f) {
        if (width[f] == 0) continue;
        // pieces of up to 16 bytes
        const int piece = std::min<int>(width[f], 16 / (int)sizeof(R));
        if (w.base[f] % piece != 0 || a.L.D % piece != 0) return -1;
        for (int st = 0; st < sets; ++st)
          if (a.stride[st] % piece != 0) return -1;
        unit = std::max(unit, piece * sizeof(R));
      }
      for (int st = 0; st < sets; ++st) {
        if (!aligned(a.x[st], unit)) return -1;
        if (backward ? !(aligned(a.dy[st], unit) && aligned(a.dx[st], unit)) : !aligned(a.y[st], unit)) return -1;
      }
      w.lanes = a.L.H * w.per;
      w.rows = kWave / w.lanes;
      return i;
    }
  }
  return -1;
}

template <bool kBackward, int NS, typename R>
int hn_lanes(int shape, const HnArgs<float, R>& a, const HnLanes& w, float* dgain, hipStream_t stream) {
  if constexpr (sizeof(R) == 4) {
    switch (shape) {
      case 0: return hn_launch_lanes<R, 2, 2, 2, NS, kBackward>(a, w, dgain, stream);
      case 1: return hn_launch_lanes<R, 4, 2, 2, NS, kBackward>(a, w, dgain, stream);
      case 2: return hn_launch_lanes<R, 4, 2, 0, NS, kBackward>(a, w, dgain, stream);
      case 3: return hn_launch_lanes<R, 2, 2, 0, NS, kBackward>(a, w, dgain, stream);
      case 4: return hn_launch_lanes<R, 4, 2, 1, NS, kBackward>(a, w, dgain, stream);
      case 5: return hn_launch_lanes<R, 4, 0, 0, NS, kBackward>(a, w, dgain, stream);
      case 6: return hn_launch_lanes<R, 0, 2, 2, NS, kBackward>(a, w, dgain, stream);
      default: return hn_launch_lanes<R, 2, 1, 1, NS, kBackward>(a, w, dgain, stream);
    }
  } else {
    switch (shape) {
      case 0: return hn_launch_lanes<R, 4, 4, 4, NS, kBackward>(a, w, dgain, stream);
      case 1: return hn_launch_lanes<R, 8, 4, 4, NS, kBackward>(a, w, dgain, stream);
      case 2: return hn_launch_lanes<R, 4, 4, 0, NS, kBackward>(a, w, dgain, stream);
      case 3: return hn_launch_lanes<R, 8, 4, 2, NS, kBackward>(a, w, dgain, stream);
      case 4: return hn_launch_lanes<R, 8, 0, 0, NS, kBackward>(a, w, dgain, stream);
      case 5: return hn_launch_lanes<R, 0, 4, 4, NS, kBackward>(a, w, dgain, stream);
      case 6: return hn_launch_lanes<R, 2, 2, 2, NS, kBackward>(a, w, dgain, stream);
      default: return hn_launch_lanes<R, 2, 1, 1, NS, kBackward>(a, w, dgain, stream);
    }
  }
}

template <bool kBackward, typename T, typename R>
int hn_dispatch(const HnArgs<T, R>& a, int sets, T* dgain, hipStream_t stream) {
  if constexpr (!std::is_same<T, double>::value) {
    HnLanes w{};
    const int shape = hn_shape(a, sets, kBackward, w);
    if (shape >= 0)
      return sets == 1 ? hn_lanes<kBackward, 1>(shape, a, w, dgain, stream)
                       : hn_lanes<kBackward, 2>(shape, a, w, dgain, stream);
    if (hn_wide(a, sets, kBackward))
      return sets == 1 ? hn_launch<T, R, 4, 1, kBackward>(a, dgain, stream)
                       : hn_launch<T, R, 4, 2, kBackward>(a, dgain, stream);
  }
  return sets == 1 ? hn_launch<T, R, 2, 1, kBackward>(a, dgain, stream)
                   : hn_launch<T, R, 2, 2, kBackward>(a, dgain, stream);
}

template <typename T, typename R>
int hn_prepare(HnArgs<T, R>& a, const R* const* x, const int64_t* strides, const T* const* gains, int64_t sets,
               const int64_t* desc, int64_t n_rows, int64_t D, int64_t F, int64_t H, const double* positions,
               const double* frequencies, int64_t axes, int64_t normalise, double eps) {
  GM_REQUIRE(sets == 1 || sets == 2, "one set of rows, or two");
  GM_REQUIRE(n_rows >= 0, "sizes must be non-negative");
  GM_REQUIRE(axes >= 0 && axes <= kHnMaxAxes, "at most 8 axes");
  const int rc = parse_heads(desc, F, H, kHnMaxHeads, D, a.L);
  if (rc != GM_OK) return rc;
  GM_REQUIRE(x && strides && gains, "the sets' pointers and strides are host arrays");
  GM_REQUIRE(!normalise || eps >= 0.0, "eps must not be negative");
  for (int f = 0; f < a.L.F; ++f) {
    a.copies += a.L.a[f];
    a.slots += a.L.n[f] == 0 ? a.L.a[f] / 2 : a.L.a[f];
    a.numbers += a.L.a[f] * (a.L.n[f] == 0 ? 1 : 2);
  }
  a.share = 1.0 / a.numbers;
  a.axes = a.slots > 0 ? (int)axes : 0;
  a.normalise = normalise != 0;
  a.n_rows = n_rows;
  a.positions = positions;
  a.frequencies = frequencies;
  a.eps = eps;
  for (int st = 0; st < sets; ++st) {
    a.x[st] = x[st];
    a.stride[st] = strides[st];
    a.gain[st] = gains[st];
    if (n_rows > 0)
      GM_REQUIRE(x[st] && (n_rows == 1 || strides[st] >= D), "rows must be device pointers, D apart or more");
  }
  if (n_rows > 0 && a.axes) GM_REQUIRE(positions && frequencies, "positions and frequencies must be device pointers");
  return GM_OK;
}

template <typename T, typename R>
int head_norm_run(const R* const* x, const int64_t* strides, const T* const* gains, int64_t sets, const int64_t* desc,
                  int64_t n_rows, int64_t D, int64_t F, int64_t H, const double* positions, const double* frequencies,
                  int64_t axes, int64_t normalise, double eps, R* const* y, void* stream) {
  HnArgs<T, R> a{};
  const int rc = hn_prepare(a, x, strides, gains, sets, desc, n_rows, D, F, H, positions, frequencies, axes, normalise,
                            eps);
  if (rc != GM_OK) return rc;
  if (n_rows == 0) return GM_OK;
  GM_REQUIRE(y, "the outputs' pointers are a host array");
  for (int st = 0; st < sets; ++st) {
    GM_REQUIRE(y[st], "outputs must be device pointers");
    a.y[st] = y[st];
  }
  return hn_dispatch<false>(a, (int)sets, (T*)nullptr, (hipStream_t)stream);
}

template <typename T, typename R>
int head_norm_back(const R* const* dy, const R* const* x, const int64_t* strides, const T* const* gains, int64_t sets,
                   const int64_t* desc, int64_t n_rows, int64_t D, int64_t F, int64_t H, const double* positions,
                   const double* frequencies, int64_t axes, int64_t normalise, double eps, R* const* dx, T* partial,
                   T* dgain, void* stream) {
  HnArgs<T, R> a{};
  const int rc = hn_prepare(a, x, strides, gains, sets, desc, n_rows, D, F, H, positions, frequencies, axes, normalise,
                            eps);
  if (rc != GM_OK) return rc;
  GM_REQUIRE(!partial == !dgain, "the gains' gradient needs its workspace");
  GM_REQUIRE(n_rows > 0, "the backward needs rows");
  GM_REQUIRE(dy && dx, "the gradients' pointers are host arrays");
  for (int st = 0; st < sets; ++st) {
    GM_REQUIRE(dy[st] && dx[st], "gradients must be device pointers");
    a.dy[st] = dy[st];
    a.dx[st] = dx[st];
  }
  a.partial = partial;
  return hn_dispatch<true>(a, (int)sets, dgain, (hipStream_t)stream);
}

}  // namespace
}  // namespace gm

extern "C" int64_t gm_head_norm_partial_rows(int64_t n_rows) {
  return n_rows < gm::kHnPartialRows ? n_rows : gm::kHnPartialRows;
}

// T: the arithmetic's type, R the rows'.
#define GM_HEAD_NORM_ENTRY(SFX, T, R)                                                                                 \
  extern "C" int gm_head_norm_forward_##SFX(const R* const* x, const int64_t* strides, const T* const* gains,         \
                                            int64_t sets, const int64_t* desc, int64_t n_rows, int64_t D, int64_t F,  \
                                            int64_t H, const double* positions, const double* frequencies,            \
                                            int64_t axes, int64_t normalise, double eps, R* const* y, void* stream) { \
    return gm::head_norm_run<T, R>(x, strides, gains, sets, desc, n_rows, D, F, H, positions, frequencies, axes,      \
                                   normalise, eps, y, stream);                                                        \
  }                                                                                                                   \
  extern "C" int gm_head_norm_backward_##SFX(                                                                         \
      const R* const* dy, const R* const* x, const int64_t* strides, const T* const* gains, int64_t sets,             \
      const int64_t* desc, int64_t n_rows, int64_t D, int64_t F, int64_t H, const double* positions,                  \
      const double* frequencies, int64_t axes, int64_t normalise, double eps, R* const* dx, T* partial, T* dgain,     \
      void* stream) {                                                                                                 \
    return gm::head_norm_back<T, R>(dy, x, strides, gains, sets, desc, n_rows, D, F, H, positions, frequencies, axes, \
                                    normalise, eps, dx, partial, dgain, stream);                                      \
  }

GM_HEAD_NORM_ENTRY(f32, float, float)
GM_HEAD_NORM_ENTRY(f64, double, double)
GM_HEAD_NORM_ENTRY(bf16, float, uint16_t)
