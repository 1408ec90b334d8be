// The differential softmax's lane kernels: a map's copies are `per_map` units of
// (A0, A1, A2) copies of frequencies 0, 1, 2, and a lane holds one unit of the query
// (the key, in the pass over sources) and reads the same unit of every row it meets,
// so that the lanes of an edge read its row as whole cache lines.  A wave's 64 lanes
// are (edge slot, unit), units rounded up to a power of two.
//
// Measured on 256x512, B = 4 (63 million edges, 40 GB of rows a pass): the forward 3.11
// ms, the passes of the backward 2.86 (targets) and 3.51 (sources).  The targets' is bound
// by its vector ALUs, busy for 91 % of the time; the sources' (62 %) and the forward (50 %
// of the time of the rows of one and four waves, 44 % of those of sixteen) by no one unit.
// The forward's rows arrive from the L1 at 23 to 24 bytes a cycle of a CU, half of the 50
// that contiguous loads reach, with the load path busy for 98 and 79 %; timing copies of it
// without the dot products take 1 % less, without the rows' loads 27 % less, without the
// records' reads from LDS nothing less, and with every source among 16 rows, all in the
// L1, 7 % less: what remains is the waves' latency, four of them a SIMD by their registers
// and the LDS of their scores (the backward, without scores, has five).  Source rows that
// neighbouring targets share are loaded for each of them: that is what would take fewer
// loads.  Fewer, wider loads did not help: a lane for both of a head's maps, five
// loads of 16 bytes for two units in place of six, took 3.1, 4.0 and 3.9 ms for the
// registers it needs; the two maps' lanes reading the pieces of up to 8 bytes together,
// each for one of two steps, 3.06, 3.0 and 3.2, and 9 % more with bfloat16 rows.
//
// Each edge's record is copied once per 64 edges into the wave's LDS (the next 64
// requested before the present ones are used) and read from there by the lanes of
// its edge.  A row of more edges than a wave's LDS holds scores of goes to four or
// sixteen waves, which combine their maxima and sums (their gradients) through LDS.
#include <algorithm>
#include <type_traits>

#include "differential.hpp"

namespace gm {
namespace {

constexpr int kDfSteps = 32;     // steps of a wave whose scores LDS holds: 32 S edges
constexpr int kDfInFlight = 4;   // the forward's steps whose rows are requested together
constexpr int kDfInFlightB = 2;  // the backward's, of which a lane reads one's gradient
constexpr int kDfThreadsB = kWavesPerBlock * kWave;
// the backward's waves a SIMD: five of float rows (the target pass of 256x512, B = 4, in 2.78 ms for 2.93 of four); with
// bfloat16 rows, whose halves take registers of their own, four (171 us against 210 of five at 64x128)
template <typename R>
constexpr int kDfWavesB = sizeof(R) == 4 ? 5 : 4;
constexpr int kDfMinLanes = 4;   // a batch of 64 edges is whole groups of those steps

struct DfUnits {
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
    for (int i = 0; i < W; ++i) v[i] = df_widen(p[i]);
  }
}
typedef __bf16 df_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t df_pack(float lo, float hi) {
  const df_bf16x2 b = {static_cast<__bf16>(lo), static_cast<__bf16>(hi)};
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
    *reinterpret_cast<uint2*>(p) = make_uint2(df_pack(v[0], v[1]), df_pack(v[2], v[3]));
  else if constexpr (W == 2)
    *reinterpret_cast<uint32_t*>(p) = df_pack(v[0], v[1]);
  else
#pragma unroll
    for (int i = 0; i < W; ++i) df_narrow(v[i], p[i]);
}

template <int A0, int A1, int A2>
struct Unit {
  static constexpr int W0 = A0, W1 = 2 * A1, W2 = 2 * A2, N = W0 + W1 + W2;
  static constexpr int NO = A2 > 0 ? 2 : 1;  // orders above 0
  static constexpr int RW = 2 + 2 * NO;      // a record's words; the sources' two more

  // A unit of node `node`'s row.  kNear: the table is below 4 GB and 2^24 rows, so a lane's place in it is a 24-bit
  // product and a 32-bit offset from a scalar address (the 64-bit form was a third of a step's instructions).
  template <bool kNear, typename R>
  static __device__ __forceinline__ void load(const R* rows, const DfUnits& w, int unit, int node, float (&v)[N]) {
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
  static __device__ __forceinline__ void store(R* row, const DfUnits& w, int unit, const float (&v)[N]) {
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
__device__ __forceinline__ Share share_of(const DfUnits& w, const int64_t* ptr) {
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

// ---------------------------------------------------------------- forward

template <typename R, int A0, int A1, int A2, bool kNear>
__global__ __launch_bounds__(1024) void differential_forward_units(DfArgs<float, R> a, DfUnits w) {
  using U = Unit<A0, A1, A2>;
  constexpr int kWords = kWave * U::RW;
  extern __shared__ __align__(16) float df_lds[];
  const Share sh = share_of(w, a.row_ptr);
  if (!sh.live) return;  // one wave a row, or the whole workgroup
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  float* rec = df_lds + sh.wave * (kWords + kDfSteps * kWave);
  float* sc = rec + kWords + lane;
  float* shared = df_lds + waves * (kWords + kDfSteps * kWave);  // (waves, 64): the waves' maxima, then sums
  const int u = lane & (w.lanes - 1), s = lane >> w.shift, unit = u < w.units ? u : w.units - 1;
  const int p = unit / w.per_map;
  const float* mine = rec + s * U::RW;  // this lane's edge of step 0
  float q[U::N];
  U::template load<false>(a.q, w, unit, sh.row, q);
  const float lambda = a.lambda[p >> 1], scale = a.scale;
  const bool second = p & 1, writes = u < w.units && unit % w.per_map == 0;
  const int held = sh.steps < kDfSteps ? sh.steps : kDfSteps;
  float m = neg_inf<float>(), l = 0.f, inv = 0.f;

  // over a lane's slots and the row's waves.  A score that is not a number is not a maximum; its exponential makes the
  // sum, and with it the row, not a number.
  auto over_waves = [&](float v, bool maximum) {
    for (int o = w.lanes; o < kWave; o <<= 1) {
      const float x = __shfl_xor(v, o, kWave);
      v = maximum ? fmaxf(x, v) : v + x;
    }
    if (sh.parts > 1) {
      __syncthreads();
      shared[sh.wave * kWave + lane] = v;
      __syncthreads();
      v = shared[lane];
      for (int o = 1; o < waves; ++o) {
        const float x = shared[o * kWave + lane];
        v = maximum ? fmaxf(x, v) : v + x;
      }
    }
    return v;
  };
  // steps t and t + 1 of the edges from `e`: the lanes of a pair of maps exchange a weight and write an edge each
  const int step = (second ? w.slots : 0) + s, ahead = writes ? step : INT32_MAX;
  const uint32_t place = (uint32_t)(step * a.L.H + (p >> 1));
  auto write = [&](int64_t e, int t, float w0, float w1) {
    const float other = other_map(second ? w0 : w1, w.per_map);
    const float v = second ? other - lambda * w1 : w0 - lambda * other;
    float* to = a.alpha + (e + t * w.slots) * a.L.H;
    if (ahead < (int)(sh.e1 - e) - t * w.slots) to[place] = v;
  };

  // phase 0: every score, its maximum; the first kDfSteps steps' stay in LDS.  The steps past them are scored again
  // for the sum (1) and the weights (2): rows beyond 16 waves' LDS only.
  for (int phase = 0; phase < 3; ++phase) {
    if (phase == 1) {
      m = over_waves(m, true);
      m = m == neg_inf<float>() ? 0.f : m;  // no edge inside: exp(-inf) = 0 everywhere
      for (int t = 0; t < held; t += 2) {  // a step past `held` is outside: its weight is zero
        const float x0 = exp2_of(sc[t * kWave] - m), x1 = exp2_of(sc[(t + 1) * kWave] - m);
        sc[t * kWave] = x0;
        sc[(t + 1) * kWave] = x1;
        l += x0 + x1;
      }
    }
    if (phase == 2) {
      l = over_waves(l, false);
      inv = l == 0.f ? 0.f : 1.f / l;
      if (a.stats && sh.part == 0 && s == 0 && writes)
        *reinterpret_cast<float2*>(a.stats + ((int64_t)sh.row * a.L.P + p) * 2) = make_float2(m, inv);
      for (int t = 0; t < held; t += 2) write(sh.e0, t, sc[t * kWave] * inv, sc[(t + 1) * kWave] * inv);
    }
    const int skip = phase == 0 ? 0 : kDfSteps;
    if (skip >= sh.steps) continue;
    const int first = skip & ~(w.lanes - 1);  // a batch's first step
    Records<U::RW> records;
    records.request(a.records, sh.e0 + (int64_t)first * w.slots, sh.e1, lane);
    for (int b = first; b < sh.steps; b += w.lanes) {
      const int64_t e = sh.e0 + (int64_t)b * w.slots;  // the batch's first edge
      wave_lds();
      records.put(rec, lane);
      wave_lds();
      if (b + w.lanes < sh.steps) records.request(a.records, e + kWave, sh.e1, lane);
      const int ends = sh.steps - b < w.lanes ? sh.steps - b : w.lanes;
      // `group` steps from t together: four in the rows of up to four waves (1.58 ms against 1.67 with two at 256x512,
      // B = 4), two in those of sixteen (1.47 against 1.53) and for the last
      auto take = [&](int t, auto group) {
        constexpr int UN = decltype(group)::value;
        float2 head[UN];
        float k[UN][U::N], cs[UN][U::NO], sn[UN][U::NO], v[UN];
#pragma unroll
        for (int n = 0; n < UN; ++n) {
          const float* r = mine + (t + n) * w.slots * U::RW;
          head[n] = *reinterpret_cast<const float2*>(r);
#pragma unroll
          for (int o = 0; o < U::NO; ++o) {
            const float2 x = *reinterpret_cast<const float2*>(r + 2 + 2 * o);
            cs[n][o] = x.x;
            sn[n][o] = x.y;
          }
        }
#pragma unroll
        for (int n = 0; n < UN; ++n) U::template load<kNear>(a.k, w, unit, __float_as_int(head[n].x), k[n]);
#pragma unroll
        for (int n = 0; n < UN; ++n) v[n] = U::dot(q, k[n], cs[n], sn[n]);
        sum_units<UN>(v, w.per_map);
#pragma unroll
        for (int n = 0; n < UN; ++n)  // outside the window: excluded, whatever its row holds
          v[n] = head[n].y == neg_inf<float>() ? neg_inf<float>() : fmaf(scale, v[n], head[n].y);
        if (phase == 0) {
#pragma unroll
          for (int n = 0; n < UN; ++n) m = fmaxf(m, v[n]);
          if (b + t < kDfSteps) {
#pragma unroll
            for (int n = 0; n < UN; ++n) sc[(b + t + n) * kWave] = v[n];
          }
        } else {
#pragma unroll
          for (int n = 0; n < UN; ++n) v[n] = exp2_of(v[n] - m);
          if (phase == 1) {
#pragma unroll
            for (int n = 0; n < UN; ++n) l += v[n];
          } else {
#pragma unroll
            for (int n = 0; n < UN; n += 2) write(e, t + n, v[n] * inv, v[n + 1] * inv);
          }
        }
      };
      int t = skip > b ? skip - b : 0;
      for (; ends - t > 2 && sh.parts <= kWavesPerBlock; t += kDfInFlight)
        take(t, std::integral_constant<int, kDfInFlight>());
      for (; t < ends; t += 2) take(t, std::integral_constant<int, 2>());
    }
  }
}

// ---------------------------------------------------------------- backward

// Sums over the wave's slots, then over a row's waves; the first wave's lanes of slot 0 hold them.
template <int M>
__device__ __forceinline__ void row_sums(const DfUnits& w, const Share& sh, float (&v)[M], float* shared) {
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

// Per target, in one walk: T = sum a g, A = sum a g tau k and B = sum a tau k, of which dq = scale c (A - T B).
template <typename R, int A0, int A1, int A2, bool kNear>
__global__ __launch_bounds__(kDfThreadsB, kDfWavesB<R>)
void differential_backward_target_units(DfArgs<float, R> a, DfUnits w) {
  using U = Unit<A0, A1, A2>;
  constexpr int kWords = kWave * U::RW, UN = kDfInFlightB, M = 2 * U::N + 1;
  extern __shared__ __align__(16) float df_lds[];
  const Share sh = share_of(w, a.row_ptr);
  if (!sh.live) return;
  const int lane = threadIdx.x & 63;
  float* rec = df_lds + sh.wave * kWords;
  const int u = lane & (w.lanes - 1), s = lane >> w.shift, unit = u < w.units ? u : w.units - 1;
  const int p = unit / w.per_map;
  const float* mine = rec + s * U::RW;
  const float scale = a.scale;
  float q[U::N];
  U::template load<false>(a.q, w, unit, sh.row, q);
  const float2 stats = *reinterpret_cast<const float2*>(a.stats + ((int64_t)sh.row * a.L.P + p) * 2);
  const bool second = p & 1;
  const int ahead = (second ? w.slots : 0) + s;
  float sums[M];
#pragma unroll
  for (int i = 0; i < M; ++i) sums[i] = 0.f;
  Records<U::RW> records;
  if (sh.steps > 0) records.request(a.records, sh.e0, sh.e1, lane);
  for (int b = 0; b < sh.steps; b += w.lanes) {
    const int64_t e = sh.e0 + (int64_t)b * w.slots;  // the batch's first edge
    wave_lds();
    records.put(rec, lane);
    wave_lds();
    if (b + w.lanes < sh.steps) records.request(a.records, e + kWave, sh.e1, lane);
    const int ends = sh.steps - b < w.lanes ? sh.steps - b : w.lanes;
    const int last = (int)(sh.e1 - e < kWave ? sh.e1 - e : kWave) - 1;  // the batch's last edge
    const float* weights = a.g + e * a.L.H;
    for (int t = 0; t < ends; t += UN) {
      float2 head[UN];
      float k[UN][U::N], cs[UN][U::NO], sn[UN][U::NO], v[UN];
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const float* r = mine + (t + n) * w.slots * U::RW;
        head[n] = *reinterpret_cast<const float2*>(r);
#pragma unroll
        for (int o = 0; o < U::NO; ++o) {
          const float2 x = *reinterpret_cast<const float2*>(r + 2 + 2 * o);
          cs[n][o] = x.x;
          sn[n][o] = x.y;
        }
      }
#pragma unroll
      for (int n = 0; n < UN; ++n) U::template load<kNear>(a.k, w, unit, __float_as_int(head[n].x), k[n]);
      // the lanes of a pair of maps read a step's gradient each
      const float held = weights[(uint32_t)(min(t * w.slots + ahead, last) * a.L.H + (p >> 1))];
#pragma unroll
      for (int n = 0; n < UN; ++n) v[n] = U::dot(q, k[n], cs[n], sn[n]);
      sum_units<UN>(v, w.per_map);
      const float other = other_map(held, w.per_map);
      const float g[UN] = {second ? other : held, second ? held : other};
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        if (head[n].y != neg_inf<float>()) {
          const float al = exp2_of(fmaf(scale, v[n], head[n].y) - stats.x), ag = al * g[n];
          U::turn(k[n], cs[n], sn[n], false);
          sums[2 * U::N] += ag;
#pragma unroll
          for (int i = 0; i < U::N; ++i) {
            sums[i] = fmaf(ag, k[n][i], sums[i]);
            sums[U::N + i] = fmaf(al, k[n][i], sums[U::N + i]);
          }
        }
      }
    }
  }
  row_sums<M>(w, sh, sums, df_lds);
  if (sh.part == 0 && s == 0 && u < w.units) {
    const float total = sums[2 * U::N] * stats.y;
    const float factor = a.gradient_scale * ((p & 1) ? -a.lambda[p >> 1] : 1.f) * stats.y;
    float dq[U::N];
#pragma unroll
    for (int i = 0; i < U::N; ++i) dq[i] = factor * (sums[i] - total * sums[U::N + i]);
    U::store(a.dq + (int64_t)sh.row * a.L.D, w, unit, dq);
    if (unit % w.per_map == 0)
      *reinterpret_cast<float3*>(a.rows + ((int64_t)sh.row * a.L.P + p) * 3) = make_float3(stats.x, stats.y, total);
  }
}

// Per source, over the edges sorted by source: dk = scale c sum a (g - T) conj(tau) q.
template <typename R, int A0, int A1, int A2, bool kNear>
__global__ __launch_bounds__(kDfThreadsB, kDfWavesB<R>)
void differential_backward_source_units(DfArgs<float, R> a, DfUnits w) {
  using U = Unit<A0, A1, A2>;
  constexpr int kRecord = U::RW + 2, kWords = kWave * kRecord, UN = kDfInFlightB;
  extern __shared__ __align__(16) float df_lds[];
  const Share sh = share_of(w, a.src_ptr);
  if (!sh.live) return;
  const int lane = threadIdx.x & 63;
  float* rec = df_lds + sh.wave * kWords;
  const int u = lane & (w.lanes - 1), s = lane >> w.shift, unit = u < w.units ? u : w.units - 1;
  const int p = unit / w.per_map;
  const float* mine = rec + s * kRecord;
  const float scale = a.scale;
  float k[U::N];
  U::template load<false>(a.k, w, unit, sh.row, k);
  float sums[U::N];
#pragma unroll
  for (int i = 0; i < U::N; ++i) sums[i] = 0.f;
  Records<kRecord> records;
  if (sh.steps > 0) records.request(a.records_s, sh.e0, sh.e1, lane);
  for (int b = 0; b < sh.steps; b += w.lanes) {
    const int64_t e = sh.e0 + (int64_t)b * w.slots;
    wave_lds();
    records.put(rec, lane);
    wave_lds();
    if (b + w.lanes < sh.steps) records.request(a.records_s, e + kWave, sh.e1, lane);
    const int ends = sh.steps - b < w.lanes ? sh.steps - b : w.lanes;
    const int left = (int)(sh.e1 - e < kWave ? sh.e1 - e : kWave);
    for (int t = 0; t < ends; t += UN) {
      float2 head[UN];
      float3 row[UN];
      float q[UN][U::N], bias[UN], cs[UN][U::NO], sn[UN][U::NO], g[UN], v[UN];
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const float* r = mine + (t + n) * w.slots * kRecord;
        const bool in = (t + n) * w.slots + s < left;  // past the row: node 0's row, edge 0's weight, excluded
        head[n] = *reinterpret_cast<const float2*>(r);
        bias[n] = r[2];
#pragma unroll
        for (int o = 0; o < U::NO; ++o) {
          const float2 x = *reinterpret_cast<const float2*>(r + 4 + 2 * o);
          cs[n][o] = x.x;
          sn[n][o] = x.y;
        }
        head[n].y = in ? head[n].y : 0.f;
        bias[n] = in ? bias[n] : neg_inf<float>();
      }
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const int i = __float_as_int(head[n].x);
        U::template load<kNear>(a.q, w, unit, i, q[n]);
        if constexpr (kNear) {
          row[n] = *reinterpret_cast<const float3*>(
              reinterpret_cast<const char*>(a.rows) +
              (__umul24((uint32_t)i, (uint32_t)(12 * a.L.P)) + 12u * (uint32_t)p));
          g[n] = *reinterpret_cast<const float*>(
              reinterpret_cast<const char*>(a.g) +
              (__float_as_uint(head[n].y) * (uint32_t)(4 * a.L.H) + 4u * (uint32_t)(p >> 1)));
        } else {
          row[n] = *reinterpret_cast<const float3*>(a.rows + ((int64_t)i * a.L.P + p) * 3);
          g[n] = a.g[(int64_t)__float_as_int(head[n].y) * a.L.H + (p >> 1)];
        }
      }
#pragma unroll
      for (int n = 0; n < UN; ++n) v[n] = U::dot(q[n], k, cs[n], sn[n]);
      sum_units<UN>(v, w.per_map);
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        if (bias[n] != neg_inf<float>()) {
          const float ds = exp2_of(fmaf(scale, v[n], bias[n]) - row[n].x) * (row[n].y * (g[n] - row[n].z));
          U::turn(q[n], cs[n], sn[n], true);
#pragma unroll
          for (int i = 0; i < U::N; ++i) sums[i] = fmaf(ds, q[n][i], sums[i]);
        }
      }
    }
  }
  row_sums<U::N>(w, sh, sums, df_lds);
  if (sh.part == 0 && s == 0 && u < w.units) {
    const float factor = a.gradient_scale * ((p & 1) ? -a.lambda[p >> 1] : 1.f);
#pragma unroll
    for (int i = 0; i < U::N; ++i) sums[i] *= factor;
    U::store(a.dk + (int64_t)sh.row * a.L.D, w, unit, sums);
  }
}

// ------------------------------------------------------------------ launch

// The unit a map's copies (a0, a1, a2) are `per_map` of, a power of two of them; the widest that serves.
struct UnitShape {
  int a0, a1, a2;
};
constexpr UnitShape kShapes[] = {{4, 2, 1}, {2, 2, 2}, {2, 2, 0}, {2, 1, 1}, {1, 1, 1}, {1, 1, 0}};
constexpr int kShapeCount = sizeof(kShapes) / sizeof(kShapes[0]);

// The shape's index and the units a map, or -1.
int find_shape(const DfLayout& L, int& per_map) {
  if (L.F < 2 || L.F > 3 || L.orders != L.F) return -1;
  for (int f = 0; f < L.F; ++f)
    if (L.n[f] != f) return -1;
  const int c[3] = {L.a[0], L.a[1], L.F == 3 ? L.a[2] : 0};
  for (int i = 0; i < kShapeCount; ++i) {
    const UnitShape& u = kShapes[i];
    if ((u.a2 == 0) != (c[2] == 0)) continue;
    for (per_map = 1; per_map * L.P <= kWave; per_map *= 2)
      if (c[0] == per_map * u.a0 && c[1] == per_map * u.a1 && c[2] == per_map * u.a2) return i;
  }
  return -1;
}

int lanes_for(int units) {
  int lanes = kDfMinLanes;
  while (lanes < units) lanes *= 2;
  return lanes;
}

// LDS words of a pass: the records a wave (and the forward's scores), or the waves' sums.
template <typename U>
size_t lds_bytes(DfPass pass, int waves, int lanes) {
  size_t words = 0;
  switch (pass) {
    case DfPass::Forward: words = (size_t)waves * (kWave * U::RW + kDfSteps * kWave + (waves > 1 ? kWave : 0)); break;
    case DfPass::BackwardTarget:
      words = (size_t)waves * std::max(kWave * U::RW, (2 * U::N + 1) * lanes);
      break;
    case DfPass::BackwardSource: words = (size_t)waves * std::max(kWave * (U::RW + 2), U::N * lanes); break;
  }
  return words * sizeof(float);
}

template <typename R, int A0, int A1, int A2, bool kNear>
int launch_shape(DfPass pass, const DfArgs<float, R>& a, DfUnits w, const DfRows& rows, hipStream_t stream) {
  using U = Unit<A0, A1, A2>;
  using Kernel = void (*)(DfArgs<float, R>, DfUnits);
  constexpr Kernel kKernels[3] = {&differential_forward_units<R, A0, A1, A2, kNear>,
                                  &differential_backward_target_units<R, A0, A1, A2, kNear>,
                                  &differential_backward_source_units<R, A0, A1, A2, kNear>};
  const Kernel kernel = kKernels[(int)pass];
  // the rows of sixteen waves; those of four and of one, in one launch of workgroups of four.  The backward holds no
  // scores, and gives the rows of sixteen four too: four workgroups a CU of as many rows, whose neighbours overlap,
  // find each other's in the L1, where one row's sixteen waves read 87 % of it from the L2 (1.21 and 1.52 ms against
  // 1.84 and 1.90 for the rows above 512 edges of 256x512, B = 4).
  const bool forward = pass == DfPass::Forward;
  w.first = 0;
  for (int c = forward ? 0 : 1; c < 2; ++c) {
    w.shared = forward ? rows.count[c] : rows.count[0] + rows.count[1];
    w.single = c == 0 ? 0 : rows.count[2];
    const int waves = c == 0 ? 16 : kWavesPerBlock;
    if (w.shared + w.single > 0) {
      const int64_t blocks = w.shared + blocks_for(w.single);
      const size_t lds = lds_bytes<U>(pass, waves, w.lanes);
      if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess)
        return check_launch("differential (LDS)");
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(waves * kWave), lds, stream, a, w);
      const int rc = check_launch("differential");
      if (rc != GM_OK) return rc;
    }
    w.first += w.shared;
  }
  return GM_OK;
}

template <bool kNear, typename R>
int launch_near(DfPass pass, int shape, const DfArgs<float, R>& a, const DfUnits& w, const DfRows& rows,
                hipStream_t stream) {
  switch (shape) {
    case 0: return launch_shape<R, 4, 2, 1, kNear>(pass, a, w, rows, stream);
    case 1: return launch_shape<R, 2, 2, 2, kNear>(pass, a, w, rows, stream);
    case 2: return launch_shape<R, 2, 2, 0, kNear>(pass, a, w, rows, stream);
    case 3: return launch_shape<R, 2, 1, 1, kNear>(pass, a, w, rows, stream);
    case 4: return launch_shape<R, 1, 1, 1, kNear>(pass, a, w, rows, stream);
    default: return launch_shape<R, 1, 1, 0, kNear>(pass, a, w, rows, stream);
  }
}

template <typename R>
int launch_units(DfPass pass, const DfArgs<float, R>& a, const DfRows& rows, hipStream_t stream) {
  DfUnits w{};
  const int shape = find_shape(a.L, w.per_map);
  if (shape < 0) return fail(GM_ERR_UNSUPPORTED, "differential: the lane kernels do not serve this layout");
  w.units = a.L.P * w.per_map;
  w.lanes = lanes_for(w.units);
  while ((1 << w.shift) < w.lanes) ++w.shift;
  w.slots = kWave / w.lanes;
  for (int f = 0; f < a.L.F; ++f) w.base[f] = a.L.off[f];
  w.row_bytes = (uint32_t)(a.L.D * sizeof(R));
  w.order = rows.order;
  const int64_t nodes = std::max(a.n_targets, a.n_sources), limit = int64_t(1) << 32;
  const bool near = nodes < (int64_t(1) << 24) && nodes * w.row_bytes < limit && nodes * a.L.P * 12 < limit &&
                    a.n_edges * a.L.H * 4 < limit;
  return near ? launch_near<true>(pass, shape, a, w, rows, stream)
              : launch_near<false>(pass, shape, a, w, rows, stream);
}

}  // namespace

// Every frequency's unit is loaded as one piece of 1, 2 or 4 numbers: the row's width and the frequency's offset are
// multiples of it (and the table's address one of 16 bytes, which the entry points check).
int df_slots(const DfLayout& L) {
  int per_map = 0;
  const int shape = find_shape(L, per_map);
  if (shape < 0) return 0;
  const UnitShape& u = kShapes[shape];
  const int width[3] = {u.a0, 2 * u.a1, 2 * u.a2};
  for (int f = 0; f < L.F; ++f)
    if (L.off[f] % width[f] != 0 || L.D % width[f] != 0) return 0;
  return kWave / lanes_for(L.P * per_map);
}

int df_launch_units(DfPass pass, const DfArgs<float, float>& a, const DfRows& rows, hipStream_t stream) {
  return launch_units<float>(pass, a, rows, stream);
}
int df_launch_units(DfPass pass, const DfArgs<float, uint16_t>& a, const DfRows& rows, hipStream_t stream) {
  return launch_units<uint16_t>(pass, a, rows, stream);
}

}  // namespace gm
