// Lanes that hold a node's units and walk its edges: a head's (a map's) copies are
// `per_map` units of (A0, A1, A2) copies of frequencies 0, 1, 2, a lane holds one
// unit of its own row and reads the same unit of every row it meets, so that the
// lanes of an edge read its row as whole cache lines.  A wave's 64 lanes are (edge
// slot, unit), units rounded up to a power of two.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace gm {

constexpr int kUnitMinLanes = 4;  // a batch of 64 edges is whole groups of four steps

__device__ __forceinline__ float row_exp2(float x) { return exp2f(x); }
__device__ __forceinline__ double row_exp2(double x) { return exp2(x); }
__device__ __forceinline__ float row_widen(float x) { return x; }
__device__ __forceinline__ double row_widen(double x) { return x; }
__device__ __forceinline__ float row_widen(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
__device__ __forceinline__ void row_narrow(float v, float& o) { o = v; }
__device__ __forceinline__ void row_narrow(double v, double& o) { o = v; }
__device__ __forceinline__ void row_narrow(float v, uint16_t& o) {  // to nearest even
  o = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
}

struct EdgeUnits {
  int units, per_map;    // lanes of an edge that hold something; units a map
  int lanes, shift;      // units rounded up to a power of two, four at least; log2
  int slots;             // 64 / lanes
  int base[3];           // the frequencies' flat offsets
  uint32_t row_bytes;
  const int32_t* order;
  // the rows of this launch, order[first ..): `shared` of all the workgroup's waves each, then `single` of one wave
  int64_t first, shared, single;
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const uint32_t lo = (uint32_t)uniform((int)(uint32_t)v), hi = (uint32_t)uniform((int)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
// A weight: one v_exp_f32 (a step off; zero below the smallest normal number).
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// The value of the lane of the head's other map, `per_map` lanes away: a DPP operand where that is the next lane, an
// LDS permute otherwise.
__device__ __forceinline__ float other_map(float v, int per_map) {
  if (per_map == 1)  // the quads' lanes 1, 0, 3, 2
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, true));
  return __shfl_xor(v, per_map, kWave);
}

// W numbers of a row at p.
template <int W>
__device__ __forceinline__ void load_w(const float* p, float* v) {
  if constexpr (W == 4) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x;
    v[1] = x.y;
    v[2] = x.z;
    v[3] = x.w;
  } else if constexpr (W == 2) {
    const float2 x = *reinterpret_cast<const float2*>(p);
    v[0] = x.x;
    v[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = p[i];
  }
}
template <int W>
__device__ __forceinline__ void load_w(const uint16_t* p, float* v) {
  if constexpr (W == 4) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(x.x << 16);
    v[1] = __uint_as_float(x.x & 0xFFFF0000u);
    v[2] = __uint_as_float(x.y << 16);
    v[3] = __uint_as_float(x.y & 0xFFFF0000u);
  } else if constexpr (W == 2) {
    const uint32_t x = *reinterpret_cast<const uint32_t*>(p);
    v[0] = __uint_as_float(x << 16);
    v[1] = __uint_as_float(x & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = row_widen(p[i]);
  }
}
typedef __bf16 row_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t row_pack(float lo, float hi) {
  const row_bf16x2 b = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
  return __builtin_bit_cast(uint32_t, b);
}
template <int W>
__device__ __forceinline__ void store_w(float* p, const float* v) {
  if constexpr (W == 4)
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else if constexpr (W == 2)
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  else
#pragma unroll
    for (int i = 0; i < W; ++i) p[i] = v[i];
}
template <int W>
__device__ __forceinline__ void store_w(uint16_t* p, const float* v) {
  if constexpr (W == 4)
    *reinterpret_cast<uint2*>(p) = make_uint2(row_pack(v[0], v[1]), row_pack(v[2], v[3]));
  else if constexpr (W == 2)
    *reinterpret_cast<uint32_t*>(p) = row_pack(v[0], v[1]);
  else
#pragma unroll
    for (int i = 0; i < W; ++i) row_narrow(v[i], p[i]);
}

template <int A0, int A1, int A2>
struct Unit {
  static constexpr int W0 = A0, W1 = 2 * A1, W2 = 2 * A2, N = W0 + W1 + W2;
  static constexpr int NO = A2 > 0 ? 2 : 1;  // orders above 0
  static constexpr int RW = 2 + 2 * NO;      // a record's words; the sources' two more

  // A unit of node `node`'s row.  kNear: the table is below 4 GB and 2^24 rows, so a lane's place in it is a 24-bit
  // product and a 32-bit offset from a scalar address (the 64-bit form was a third of a step's instructions).
  template <bool kNear, typename R>
  static __device__ __forceinline__ void load(const R* rows, const EdgeUnits& w, int unit, int node, float (&v)[N]) {
    if constexpr (kNear) {
      const uint32_t row = __umul24((uint32_t)node, w.row_bytes);
      auto at = [&](int f, int width) {
        return reinterpret_cast<const R*>(reinterpret_cast<const char*>(rows + w.base[f]) +
                                          (row + (uint32_t)(unit * width) * (uint32_t)sizeof(R)));
      };
      load_w<W0>(at(0, W0), v);
      load_w<W1>(at(1, W1), v + W0);
      if constexpr (W2 > 0) load_w<W2>(at(2, W2), v + W0 + W1);
    } else {
      const R* row = reinterpret_cast<const R*>(reinterpret_cast<const char*>(rows) + (int64_t)node * w.row_bytes);
      load_w<W0>(row + w.base[0] + unit * W0, v);
      load_w<W1>(row + w.base[1] + unit * W1, v + W0);
      if constexpr (W2 > 0) load_w<W2>(row + w.base[2] + unit * W2, v + W0 + W1);
    }
  }
  template <typename R>
  static __device__ __forceinline__ void store(R* row, const EdgeUnits& w, int unit, const float (&v)[N]) {
    store_w<W0>(row + w.base[0] + unit * W0, v);
    store_w<W1>(row + w.base[1] + unit * W1, v + W0);
    if constexpr (W2 > 0) store_w<W2>(row + w.base[2] + unit * W2, v + W0 + W1);
  }
  // The three passes form a weight by the same roundings, so that a row's ds sum to zero as nearly as its weights to one:
  // a key bias's gradient, zero but for rounding, is a third smaller than with the gathered row turned before the dot in
  // the backward's passes (which saves a fifth of their instructions and 1 % of their time).
  // Re< q, tau k >: per order cos sum (q0 k0 + q1 k1) + sin sum (q1 k0 - q0 k1)
  static __device__ __forceinline__ float dot(const float (&q)[N], const float (&k)[N], const float (&cs)[NO],
                                              const float (&sn)[NO]) {
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < W0; ++i) acc = fmaf(q[i], k[i], acc);
#pragma unroll
    for (int o = 0; o < NO; ++o) {
      const int at = o == 0 ? W0 : W0 + W1, width = o == 0 ? W1 : W2;
      float re = 0.f, im = 0.f;
#pragma unroll
      for (int i = 0; i < width; i += 2) {
        re = fmaf(q[at + i], k[at + i], fmaf(q[at + i + 1], k[at + i + 1], re));
        im = fmaf(q[at + i + 1], k[at + i], fmaf(-q[at + i], k[at + i + 1], im));
      }
      acc = fmaf(cs[o], re, fmaf(sn[o], im, acc));
    }
    return acc;
  }
  // tau k, or with `back` conj(tau) k, in place
  static __device__ __forceinline__ void turn(float (&k)[N], const float (&cs)[NO], const float (&sn)[NO], bool back) {
#pragma unroll
    for (int o = 0; o < NO; ++o) {
      const int at = o == 0 ? W0 : W0 + W1, width = o == 0 ? W1 : W2;
      const float s = back ? -sn[o] : sn[o];
#pragma unroll
      for (int i = 0; i < width; i += 2) {
        const float k0 = k[at + i], k1 = k[at + i + 1];
        k[at + i] = cs[o] * k0 - s * k1;
        k[at + i + 1] = cs[o] * k1 + s * k0;
      }
    }
  }
};

// One wave's records of 64 edges: `words` a record, in flight a batch ahead.
template <int WORDS>
struct Records {
  static constexpr int kLoads = WORDS / 2;
  float2 next[kLoads];
  // request the records of edges [base, min(base + 64, end)); past them: edges of node 0 outside the window
  __device__ __forceinline__ void request(const float* records, int64_t base, int64_t end, int lane) {
    const int64_t left = end - base;
    const int pieces = (int)(left < kWave ? left : kWave) * kLoads;
    const float2* from = reinterpret_cast<const float2*>(records + base * WORDS);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = i * kWave + lane;
      next[i] = at < pieces ? from[at] : make_float2(0.f, neg_inf<float>());
    }
  }
  __device__ __forceinline__ void put(float* lds, int lane) const {
    float2* to = reinterpret_cast<float2*>(lds);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) to[i * kWave + lane] = next[i];
  }
};

// The wave's LDS writes are seen by its other lanes' reads, and the reads before them are done.
__device__ __forceinline__ void wave_lds() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A map's units added, for the steps at hand.
template <int UN>
__device__ __forceinline__ void sum_units(float (&v)[UN], int per_map) {
  if (per_map > 1) {
    for (int o = 1; o < per_map; o <<= 1) {
#pragma unroll
      for (int n = 0; n < UN; ++n) v[n] += __shfl_xor(v[n], o, kWave);
    }
  }
}

// Which row a wave works on, and which of its edges; all of it scalar.
struct Share {
  int64_t e0, e1;  // this wave's edges
  int row, wave, part, parts, steps;  // parts: the row's waves
  bool live;
};
__device__ __forceinline__ Share share_of(const EdgeUnits& w, const int64_t* ptr) {
  Share s;
  s.wave = uniform((int)(threadIdx.x >> 6));
  const int waves = blockDim.x >> 6;
  const bool one = blockIdx.x >= w.shared;
  const int64_t at = one ? w.shared + xcd_spread_block(blockIdx.x - w.shared, gridDim.x - w.shared) * waves + s.wave
                         : xcd_spread_block(blockIdx.x, w.shared);
  s.part = one ? 0 : s.wave;
  s.parts = one ? 1 : waves;
  s.live = at < w.shared + w.single;
  s.row = s.live ? uniform((int)w.order[w.first + at]) : 0;
  const int64_t e0 = s.live ? uniform(ptr[s.row]) : 0, e1 = s.live ? uniform(ptr[s.row + 1]) : 0;
  const int64_t steps = (e1 - e0 + w.slots - 1) >> (6 - w.shift);
  const int64_t per = (one ? steps : (steps + waves - 1) / waves) << (6 - w.shift);
  s.e0 = e0 + s.part * per < e1 ? e0 + s.part * per : e1;
  s.e1 = s.e0 + per < e1 ? s.e0 + per : e1;
  s.steps = (int)((s.e1 - s.e0 + w.slots - 1) >> (6 - w.shift));
  return s;
}

// Sums over the wave's slots, then over a row's waves; the first wave's lanes of slot 0 hold them.
template <int M>
__device__ __forceinline__ void row_sums(const EdgeUnits& w, const Share& sh, float (&v)[M], float* shared) {
  const int lane = threadIdx.x & 63, wave = sh.wave;
  for (int o = w.lanes; o < kWave; o <<= 1) {
#pragma unroll
    for (int i = 0; i < M; ++i) v[i] += __shfl_xor(v[i], o, kWave);
  }
  if (sh.parts == 1) return;
  __syncthreads();  // the records have been read
  if (lane < w.lanes) {
#pragma unroll
    for (int i = 0; i < M; ++i) shared[(wave * M + i) * w.lanes + lane] = v[i];
  }
  __syncthreads();
  if (wave == 0 && lane < w.lanes) {
    for (int o = 1; o < sh.parts; ++o)
#pragma unroll
      for (int i = 0; i < M; ++i) v[i] += shared[(o * M + i) * w.lanes + lane];
  }
}

inline int lanes_for(int units) {
  int lanes = kUnitMinLanes;
  while (lanes < units) lanes *= 2;
  return lanes;
}

}  // namespace gm
