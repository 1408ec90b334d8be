// The lane kernels of the softmax with a learned relative bias: a head's copies are
// `per_map` units of (A0, A1, A2) copies of frequencies 0, 1, 2, one lane a unit
// (edge_units.hpp), so that a step of a wave takes S = 64 / lanes edges.
//
// Forward, a wave a target (a long row four): a step gathers S rows of k and sums a
// score over its units' lanes; scores wait in LDS (a long row's in alpha) for their
// maximum and sum.  63.0 M edges of 160 numbers take 2.67 ms: rows reach a CU out of L1
// at 27 bytes a cycle (contiguous loads at 50) while vector instructions fill half of the
// time, and neither gives way alone (at 2.83 ms: all rows among 16 nodes 6% less, without
// the dots 2%, without the weights' writes 8%).
//
// Backward, dq and dk: a wave a pair of neighbouring rows over the nodes of both, whose
// rows are loaded once for two edges (four loads for seven edges on a grid).  1.76 and
// 1.82 ms for the edges above; a row at a time 2.50 and 2.64.  Scores do not gain from
// pairs (3.68 ms): twice the registers of q, entries of 56 bytes, and alpha's places edge
// by edge cost more than the rows' loads they spare.
#pragma once
#include <algorithm>
#include <type_traits>

#include "edge_units.hpp"
#include "relative.hpp"

namespace gm {
namespace rel {

constexpr int kRelKept = 16;  // rows of scores that LDS holds a wave: 16 steps, or 32 where two lanes share a head's
// Steps whose rows are requested together: two, and the registers that this leaves go to more waves, five or six a SIMD
// (four steps and four waves took 9 % more for the scores of 33 M edges, 16 % for the rows of 63 M).
constexpr int kRelInFlight = 2;
constexpr int kRelThreads = kWavesPerBlock * kWave;
// What stands among a row's exponentials for a score of -inf, outside the window for one: no exponential has these
// bits, and as a number they add nothing.  Its weight is zero in any row, one whose sum is no number too.
constexpr uint32_t kRelNone = 0x80000000u;

// A lane's shape; NO, the orders of the tables above 0.
template <int A0, int A1, int A2, int ORD>
struct RelUnit {
  static constexpr int W0 = A0, W1 = 2 * A1, W2 = 2 * A2, N = W0 + W1 + W2;
  static constexpr int NO = ORD;
  static constexpr int RW = 2 + 2 * NO;                     // words of an edge's record
  static constexpr int PW = kRelPairHead + 4 * NO;          // of a pair's entry
  static constexpr int NA = NO > 0 ? NO : 1;  // arrays of none

  template <bool kNear, typename R>
  static __device__ __forceinline__ void load(const R* rows, const EdgeUnits& w, int unit, int node, float (&v)[N]) {
    if constexpr (kNear) {
      const uint32_t row = __umul24((uint32_t)node, w.row_bytes);
      auto at = [&](int f, int width) {
        return reinterpret_cast<const R*>(reinterpret_cast<const char*>(rows + w.base[f]) +
                                          (row + (uint32_t)(unit * width) * (uint32_t)sizeof(R)));
      };
      if constexpr (W0 > 0) load_w<W0>(at(0, W0), v);
      if constexpr (W1 > 0) load_w<W1>(at(1, W1), v + W0);
      if constexpr (W2 > 0) load_w<W2>(at(2, W2), v + W0 + W1);
    } else {
      const R* row = reinterpret_cast<const R*>(reinterpret_cast<const char*>(rows) + (int64_t)node * w.row_bytes);
      if constexpr (W0 > 0) load_w<W0>(row + w.base[0] + unit * W0, v);
      if constexpr (W1 > 0) load_w<W1>(row + w.base[1] + unit * W1, v + W0);
      if constexpr (W2 > 0) load_w<W2>(row + w.base[2] + unit * W2, v + W0 + W1);
    }
  }
  template <typename R>
  static __device__ __forceinline__ void store(R* row, const EdgeUnits& w, int unit, const float (&v)[N]) {
    if constexpr (W0 > 0) store_w<W0>(row + w.base[0] + unit * W0, v);
    if constexpr (W1 > 0) store_w<W1>(row + w.base[1] + unit * W1, v + W0);
    if constexpr (W2 > 0) store_w<W2>(row + w.base[2] + unit * W2, v + W0 + W1);
  }
  // (cos, sin) of an entry's edge j, whose pairs lie order by order, (cos, sin) of both edges each
  static __device__ __forceinline__ void phases(const float* r, int j, float (&cs)[NA], float (&sn)[NA]) {
#pragma unroll
    for (int o = 0; o < NO; ++o) {
      const float2 x = *reinterpret_cast<const float2*>(r + 4 * o + 2 * j);
      cs[o] = x.x;
      sn[o] = x.y;
    }
  }
  // the frequency of order o + 1's numbers: where they start, how many
  static constexpr int start(int o) { return o == 0 ? W0 : W0 + W1; }
  static constexpr int width(int o) { return o == 0 ? W1 : W2; }

  // Re< q, tau k >: per order cos sum (q0 k0 + q1 k1) + sin sum (q1 k0 - q0 k1)
  static __device__ __forceinline__ float dot(const float (&q)[N], const float (&k)[N], const float (&cs)[NA],
                                              const float (&sn)[NA]) {
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < W0; ++i) acc = fmaf(q[i], k[i], acc);
#pragma unroll
    for (int o = 0; o < NO; ++o) {
      float re = 0.f, im = 0.f;
#pragma unroll
      for (int i = 0; i < width(o); i += 2) {
        const int at = start(o) + i;
        re = fmaf(q[at], k[at], fmaf(q[at + 1], k[at + 1], re));
        im = fmaf(q[at + 1], k[at], fmaf(-q[at], k[at + 1], im));
      }
      if (width(o) > 0) acc = fmaf(cs[o], re, fmaf(sn[o], im, acc));
    }
    return acc;
  }
  // sums += d tau k, or with `back` d conj(tau) k
  static __device__ __forceinline__ void add(float* sums, float d, const float (&k)[N], const float (&cs)[NA],
                                             const float (&sn)[NA], bool back) {
#pragma unroll
    for (int i = 0; i < W0; ++i) sums[i] = fmaf(d, k[i], sums[i]);
#pragma unroll
    for (int o = 0; o < NO; ++o) {
      const float c = d * cs[o], s = back ? -d * sn[o] : d * sn[o];
#pragma unroll
      for (int i = 0; i < width(o); i += 2) {
        const int at = start(o) + i;
        sums[at] = fmaf(c, k[at], fmaf(-s, k[at + 1], sums[at]));
        sums[at + 1] = fmaf(c, k[at + 1], fmaf(s, k[at], sums[at + 1]));
      }
    }
  }
};

// The value of the neighbouring lane, which holds the other step of a pair for the same head: a DPP operand.
__device__ __forceinline__ float next_lane(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xB1, 0xF, 0xF, true));
}

// The row (a target, or a pair) that a wave works on, and which of its edges or entries; all of it scalar.
__device__ __forceinline__ Share rel_share(const EdgeUnits& w, const int64_t* ptr) {
  constexpr int waves = kWavesPerBlock;
  Share s;
  s.wave = uniform((int)(threadIdx.x >> 6));
  const uint32_t block = blockIdx.x, shared = (uint32_t)w.shared;
  const bool one = block >= shared;
  const uint32_t spread = xcd_spread_block32(one ? block - shared : block, one ? gridDim.x - shared : shared);
  const int64_t at = one ? shared + (int64_t)spread * waves + s.wave : spread;
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

// kSplit: a head has two units or more, whose lanes hold the same scores: two of them keep every second step's each.
template <typename R, typename U, bool kNear, bool kSplit>
__global__ __launch_bounds__(kRelThreads, 5) void relative_forward_units(RelArgs<float, R> a, EdgeUnits w) {
  constexpr int kWords = kWave * U::RW, kEvery = kSplit ? 2 : 1;  // steps of a row of scores, of which a lane keeps one
  extern __shared__ __align__(16) float rel_lds[];
  const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6)), H = a.L.H;
  float* rec = rel_lds + wave * (kWords + kRelKept * kWave);
  float* sc = rec + kWords + lane;
  float* shared = rel_lds + kWavesPerBlock * (kWords + kRelKept * kWave);  // (waves, 64): the waves' maxima, then sums
  float* learned = shared + kWavesPerBlock * kWave;                        // (buckets, H), in units of log 2
  for (int i = threadIdx.x; i < a.buckets * H; i += blockDim.x) learned[i] = a.table[i] * (float)kRelLog2e;
  __syncthreads();
  const int u = lane & (w.lanes - 1), s = lane >> w.shift, unit = u < w.units ? u : w.units - 1;
  const int per = __builtin_ctz(w.per_map), h = unit >> per, own = unit & (w.per_map - 1);  // powers of two
  const int odd = kSplit ? own & 1 : 0;
  const float* mine = rec + s * U::RW;  // this lane's edge of step 0
  const float scale = a.scale;
  const float* bias_of = learned + h;

  const Share sh = rel_share(w, a.row_ptr);
  if (!sh.live) return;  // one wave a row, or the whole workgroup
  float q[U::N];
  U::template load<false>(a.q, w, unit, sh.row, q);
  float m = neg_inf<float>(), l = 0.f;

  // over a lane's slots (and the two lanes with a step each) and the row's waves.  A score that is not a number is not
  // a maximum; its exponential makes the sum, and with it the row, not a number.
  auto over_waves = [&](float v, bool maximum) {
    for (int o = w.lanes; o < kWave; o <<= 1) {
      const float x = __shfl_xor(v, o, kWave);
      v = maximum ? fmaxf(x, v) : v + x;
    }
    if constexpr (kSplit) {
      const float x = next_lane(v);
      v = maximum ? fmaxf(x, v) : v + x;
    }
    if (sh.parts > 1) {
      __syncthreads();
      shared[sh.wave * kWave + lane] = v;
      __syncthreads();
      v = shared[lane];
      for (int o = 1; o < kWavesPerBlock; ++o) {
        const float x = shared[o * kWave + lane];
        v = maximum ? fmaxf(x, v) : v + x;
      }
    }
    return v;
  };

  // The scores: the first kRelKept rows stay in LDS, those past them wait in alpha.  A row's numbers lie side by side
  // there, and lane after lane writes and reads them, `from` the lane that formed them (whose own place is lane `to`'s):
  // a lane's own places alternate between two steps (2.77 ms for 2.73, and a fifth more accesses to L1).
  const int rows = (sh.steps + kEvery - 1) / kEvery, held = rows < kRelKept ? rows : kRelKept;
  const int numbers = kEvery * w.slots * H, edge = (int)((uint32_t)lane * a.by_heads >> 16);  // lane / H
  const int step = edge >> (6 - w.shift), slot = edge & (w.slots - 1);
  const int from = lane < numbers ? slot * w.lanes + ((lane - edge * H) << per) + step : lane;
  const int to = own < kEvery && u < w.units ? (odd * w.slots + s) * H + h : lane;
  // a lane's rows: all but the last for all lanes, the last for those within the row's edges
  const int last = (int)((sh.e1 - sh.e0) * H - (int64_t)(rows - 1) * numbers);
  const int mine_rows = lane < numbers ? (lane < last ? rows : rows - 1) : 0;
  auto has = [&](int r) { return r < mine_rows; };
  auto out = [&](int r) -> float& { return (a.alpha + (sh.e0 * H + (int64_t)r * numbers))[(uint32_t)lane]; };

  Records<U::RW> records;
  if (sh.steps > 0) records.request(a.records, sh.e0, sh.e1, lane);
  for (int b = 0; b < sh.steps; b += w.lanes) {
    const int64_t e = sh.e0 + (int64_t)b * w.slots;  // the batch's first edge
    wave_lds();
    records.put(rec, lane);
    wave_lds();
    if (b + w.lanes < sh.steps) records.request(a.records, e + kWave, sh.e1, lane);
    const int ends = sh.steps - b < w.lanes ? sh.steps - b : w.lanes;
    auto take = [&](int t, auto group) {
      constexpr int UN = decltype(group)::value;
      float k[UN][U::N], cs[UN][U::NA], sn[UN][U::NA], v[kRelInFlight] = {};
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const float* r = mine + (t + n) * w.slots * U::RW;
        U::template load<kNear>(a.k, w, unit, __float_as_int(r[0]) & 0xFFFFFF, k[n]);
#pragma unroll
        for (int o = 0; o < U::NO; ++o) {
          const float2 x = *reinterpret_cast<const float2*>(r + 2 + 2 * o);
          cs[n][o] = x.x;
          sn[n][o] = x.y;
        }
      }
#pragma unroll
      for (int n = 0; n < UN; ++n) v[n] = U::dot(q, k[n], cs[n], sn[n]);
#pragma unroll
      for (int n = 0; n < UN; n += kEvery) {  // a step past the row's last is outside the window
        const float2 head = *reinterpret_cast<const float2*>(mine + (t + n + odd) * w.slots * U::RW);
        float x = v[n];
        if constexpr (kSplit) {  // an even lane keeps the first step's sum, an odd one the second's
          const float keep = odd ? v[n + 1] : v[n], give = odd ? v[n] : v[n + 1];
          x = keep + next_lane(give);
          for (int o = 2; o < w.per_map; o <<= 1) x += __shfl_xor(x, o, kWave);
        }
        // outside the window: excluded, whatever its row holds
        x = head.y == neg_inf<float>() ? neg_inf<float>()
                                       : fmaf(scale, x, head.y + bias_of[__umul24(__float_as_uint(head.x) >> 24, (uint32_t)H)]);
        const int r = (b + t + n) / kEvery;
        m = fmaxf(m, x);
        if (r < kRelKept) {
          sc[r * kWave] = x;
        } else {
          const float y = __shfl(x, from, kWave);
          if (has(r)) out(r) = y;
        }
      }
    };
    int t = 0;
    for (; t + kRelInFlight <= ends; t += kRelInFlight) take(t, std::integral_constant<int, kRelInFlight>());
    if (t < ends) take(t, std::integral_constant<int, 1>());
  }
  m = over_waves(m, true);
  m = m == neg_inf<float>() ? 0.f : m;  // no edge inside: exp(-inf) = 0 everywhere
  for (int r = 0; r < held; ++r) {
    const float score = sc[r * kWave], x = exp2_of(score - m);
    sc[r * kWave] = score == neg_inf<float>() ? __uint_as_float(kRelNone) : x;
    l += x;
  }
  if (rows > kRelKept) {
    const float top = __shfl(m, from, kWave);
    float sum = 0.f;
#pragma unroll 4
    for (int r = kRelKept; r < rows; ++r) sum += has(r) ? exp2_of(out(r) - top) : 0.f;
    l += __shfl(sum, to, kWave);
  }
  l = over_waves(l, false);
  const float inv = __shfl(l == 0.f ? 0.f : 1.f / l, from, kWave);
  wave_lds();
  const float* formed = sc - lane + from;
  for (int r = 0; r < held; ++r) {
    const float x = formed[r * kWave];
    if (has(r)) out(r) = __float_as_uint(x) == kRelNone ? 0.f : x * inv;
  }
  if (rows > kRelKept) {
    const float top = __shfl(m, from, kWave);
#pragma unroll 4
    for (int r = kRelKept; r < rows; ++r) {
      if (!has(r)) continue;
      const float score = out(r);
      out(r) = score == neg_inf<float>() ? 0.f : exp2_of(score - top) * inv;
    }
  }
}

// ---------------------------------------------------------------- backward

// Per pair of targets or of sources (kTargets or not): dq = scale sum ds tau k over a target's edges, dk = scale sum ds
// conj(tau) q over a source's.
template <typename R, typename U, bool kNear, bool kTargets, bool kSplit>
__global__ __launch_bounds__(kRelThreads, (U::N > 10 ? 5 : 6)) void relative_rows_units(RelArgs<float, R> a,
                                                                                         EdgeUnits w) {
  constexpr int RW = U::PW, kWords = kWave * RW;
  constexpr int kT = kSplit ? 1 : 2;
  extern __shared__ __align__(16) float rel_lds[];
  const Share sh = rel_share(w, kTargets ? a.pair_ptr : a.pair_ptr_s);
  if (!sh.live) return;
  const int lane = threadIdx.x & 63, H = a.L.H;
  float* rec = rel_lds + sh.wave * kWords;
  const int u = lane & (w.lanes - 1), s = lane >> w.shift, unit = u < w.units ? u : w.units - 1;
  const int h = unit >> __builtin_ctz(w.per_map), odd = kSplit ? unit & 1 : 0;  // units a head: a power of two
  const float* mine = rec + s * RW;
  const float* records_of = kTargets ? a.pairs : a.pairs_s;
  float sums[2 * U::N];
#pragma unroll
  for (int i = 0; i < 2 * U::N; ++i) sums[i] = 0.f;
  Records<RW> records;
  if (sh.steps > 0) records.request(records_of, sh.e0, sh.e1, lane);
  for (int b = 0; b < sh.steps; b += w.lanes) {
    const int64_t e = sh.e0 + (int64_t)b * w.slots;
    wave_lds();
    records.put(rec, lane);
    wave_lds();
    if (b + w.lanes < sh.steps) records.request(records_of, e + kWave, sh.e1, lane);
    const int ends = sh.steps - b < w.lanes ? sh.steps - b : w.lanes;
    auto take = [&](int t, auto group) {
      constexpr int UN = decltype(group)::value;
      float x[UN][U::N], d[UN][kT];
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const float* r = mine + (t + n) * w.slots * RW;
#pragma unroll
        for (int j = 0; j < kT; ++j) {
          const int edge = __float_as_int(r[1 + 2 * (odd + j)]);  // past the end: negative
          const uint32_t place = edge < 0 ? 0u : (uint32_t)edge;
          float ds;
          if constexpr (kNear)  // as the rows': a 32-bit offset from a scalar address
            ds = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(a.ds) +
                                                 (place * (uint32_t)(4 * H) + 4u * (uint32_t)h));
          else
            ds = a.ds[(int64_t)place * H + h];
          d[n][j] = edge < 0 ? 0.f : ds;
        }
        U::template load<kNear>(kTargets ? a.k : a.q, w, unit, __float_as_int(r[0]), x[n]);
      }
#pragma unroll
      for (int n = 0; n < UN; ++n) {
        const float* r = mine + (t + n) * w.slots * RW;
        float both[2];
        if constexpr (kSplit) {  // an even lane has the first row's, an odd one the second's
          const float other = next_lane(d[n][0]);
          both[0] = odd ? other : d[n][0];
          both[1] = odd ? d[n][0] : other;
        } else {
          both[0] = d[n][0];
          both[1] = d[n][kT - 1];
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (both[j] != 0.f) {
            float cs[U::NA], sn[U::NA];
            U::phases(r + kRelPairHead, j, cs, sn);
            U::add(sums + j * U::N, both[j], x[n], cs, sn, !kTargets);
          }
        }
      }
    };
    int t = 0;
    for (; t + kRelInFlight <= ends; t += kRelInFlight) take(t, std::integral_constant<int, kRelInFlight>());
    if (t < ends) take(t, std::integral_constant<int, 1>());
  }
  row_sums<2 * U::N>(w, sh, sums, rel_lds);
  if (sh.part == 0 && s == 0 && u < w.units) {
    R* rows = kTargets ? a.dq : a.dk;
    const int64_t count = kTargets ? a.n_targets : a.n_sources;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t row = 2 * (int64_t)sh.row + j;
      float v[U::N];
#pragma unroll
      for (int i = 0; i < U::N; ++i) v[i] = a.gradient_scale * sums[j * U::N + i];
      if (row < count) U::store(rows + row * a.L.D, w, unit, v);
    }
  }
}

// ------------------------------------------------------------------ launch

// The unit a head's copies (a0, a1, a2) are `per_map` of, a power of two of them; the widest that serves.
struct RelShape {
  int a0, a1, a2;
};
constexpr RelShape kRelShapes[] = {{4, 2, 2}, {4, 2, 1}, {2, 2, 2}, {2, 1, 1}, {1, 1, 1},
                                   {2, 2, 0}, {1, 1, 0}, {4, 0, 0}, {1, 0, 0}, {0, 2, 2}, {0, 1, 1}};
constexpr int kRelShapeCount = sizeof(kRelShapes) / sizeof(kRelShapes[0]);

// A head's copies at frequencies 0, 1, 2; false where there are others, or the tables hold more orders than that.
inline bool rel_copies(const RelLayout& L, int (&c)[3], int (&base)[3]) {
  for (int f = 0; f < 3; ++f) c[f] = base[f] = 0;
  for (int f = 0; f < L.F; ++f) {
    if (L.n[f] > 2) return false;
    c[L.n[f]] = L.a[f];
    base[L.n[f]] = L.off[f];
  }
  return L.orders == (c[2] > 0 ? 3 : (c[1] > 0 ? 2 : 1));
}

// The shape's index and the units a head, or -1.
inline int rel_shape(const RelLayout& L, int& per_map, int (&base)[3]) {
  int c[3];
  if (!rel_copies(L, c, base)) return -1;
  for (int i = 0; i < kRelShapeCount; ++i) {
    const RelShape& u = kRelShapes[i];
    for (per_map = 1; per_map * L.H <= kWave; per_map *= 2)
      if (c[0] == per_map * u.a0 && c[1] == per_map * u.a1 && c[2] == per_map * u.a2) return i;
  }
  return -1;
}

// LDS of a pass: the records a wave (and the forward's scores, the waves' maxima and the learned table), the waves'
// sums: at most 39 KB forward (256 buckets of 16 heads) and 24 KB backward, of the 64 KB that any launch may ask for.
template <typename U>
size_t rel_forward_lds(int table) {
  return sizeof(float) * ((size_t)kWavesPerBlock * kWave * (U::RW + kRelKept + 1) + table);
}
template <typename U>
size_t rel_rows_lds(int lanes) {
  return sizeof(float) * kWavesPerBlock * (size_t)std::max(kWave * U::PW, 2 * U::N * lanes);
}

template <typename R, typename U, bool kNear, bool kSplit>
int rel_launch(RelPass pass, const RelArgs<float, R>& a, EdgeUnits w, const RelRows& rows, hipStream_t stream) {
  w.first = 0;
  w.shared = rows.count[0] + rows.count[1];
  w.single = rows.count[2];
  const int64_t blocks = w.shared + blocks_for(w.single);
  if (blocks == 0) return GM_OK;
  const auto kernel = pass == RelPass::Forward          ? &relative_forward_units<R, U, kNear, kSplit>
                      : pass == RelPass::BackwardTarget ? &relative_rows_units<R, U, kNear, true, kSplit>
                                                        : &relative_rows_units<R, U, kNear, false, kSplit>;
  const size_t lds = pass == RelPass::Forward ? rel_forward_lds<U>(a.buckets * a.L.H) : rel_rows_lds<U>(w.lanes);
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kRelThreads), lds, stream, a, w);
  return check_launch("relative");
}

template <typename R, int A0, int A1, int A2>
int rel_launch_shape(RelPass pass, const RelArgs<float, R>& a, const EdgeUnits& w, const RelRows& rows, bool near,
                     hipStream_t stream) {
  using U = RelUnit<A0, A1, A2, (A2 > 0 ? 2 : (A1 > 0 ? 1 : 0))>;
  if (near)
    return w.per_map > 1 ? rel_launch<R, U, true, true>(pass, a, w, rows, stream)
                         : rel_launch<R, U, true, false>(pass, a, w, rows, stream);
  return w.per_map > 1 ? rel_launch<R, U, false, true>(pass, a, w, rows, stream)
                       : rel_launch<R, U, false, false>(pass, a, w, rows, stream);
}

template <typename R>
int rel_launch_any(RelPass pass, const RelArgs<float, R>& a, const RelRows& rows, hipStream_t stream) {
  EdgeUnits w{};
  const int shape = rel_shape(a.L, w.per_map, w.base);
  if (shape < 0) return fail(GM_ERR_UNSUPPORTED, "relative: the lane kernels do not serve this layout");
  w.units = a.L.H * w.per_map;
  w.lanes = lanes_for(w.units);
  while ((1 << w.shift) < w.lanes) ++w.shift;
  w.slots = kWave / w.lanes;
  w.row_bytes = (uint32_t)(a.L.D * sizeof(R));
  w.order = rows.order;
  const int64_t nodes = std::max(a.n_targets, a.n_sources), limit = int64_t(1) << 32;
  const bool near = nodes <= (int64_t(1) << 24) && nodes * w.row_bytes < limit && a.n_edges * a.L.H * 4 < limit;
  switch (shape) {
    case 0: return rel_launch_shape<R, 4, 2, 2>(pass, a, w, rows, near, stream);
    case 1: return rel_launch_shape<R, 4, 2, 1>(pass, a, w, rows, near, stream);
    case 2: return rel_launch_shape<R, 2, 2, 2>(pass, a, w, rows, near, stream);
    case 3: return rel_launch_shape<R, 2, 1, 1>(pass, a, w, rows, near, stream);
    case 4: return rel_launch_shape<R, 1, 1, 1>(pass, a, w, rows, near, stream);
    case 5: return rel_launch_shape<R, 2, 2, 0>(pass, a, w, rows, near, stream);
    case 6: return rel_launch_shape<R, 1, 1, 0>(pass, a, w, rows, near, stream);
    case 7: return rel_launch_shape<R, 4, 0, 0>(pass, a, w, rows, near, stream);
    case 8: return rel_launch_shape<R, 1, 0, 0>(pass, a, w, rows, near, stream);
    case 9: return rel_launch_shape<R, 0, 2, 2>(pass, a, w, rows, near, stream);
    default: return rel_launch_shape<R, 0, 1, 1>(pass, a, w, rows, near, stream);
  }
}

}  // namespace rel
}  // namespace gm
