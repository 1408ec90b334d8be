// The neighbourhood softmax with a learned relative bias over CSR neighbour lists,
// forward and backward.  Per edge e = (i <- j) in bucket b(e) and head h:
//   s_h   = scale sum_n Re< q_i,n,h , tau_n(e) k_j,n,h > + bias(e) + table[b(e), h]
//   alpha = softmax of s_h over i's edges inside the window (zero outside; a target
//           with no edge inside has only zeros)
// and from g = d alpha, with T_h(i) = sum_e alpha g:
//   ds = alpha (g - T),   dtable[b, h] = sum of ds over the edges of bucket b
//   dq_i = scale sum_e ds tau k_j,   dk_j = scale sum_e ds conj(tau) q_i
//
// The backward reads the forward's weights: a score is formed once.  A pass over
// alpha and g, which lie edge by edge, writes ds and adds the buckets' sums; one over
// the targets and one over the sources read ds.  An edge of weight zero counts for
// nothing, whatever its rows and its g hold: so do the edges outside the window.  No
// atomics between waves: sums are in a fixed order.
//
// Per edge a pass reads one record of 32-bit words (64-bit for double): the source
// with the bucket above it, the bias in units of log 2 (-inf outside the window) and
// the transport's (cos, sin) of orders 1 .., packed once for an edge set; the source
// side's name the target and the edge.  (The backward's lane kernels read the merged
// entries of two rows instead: relative.hpp.)
#include "relative.hpp"
#include "partial_sum.hpp"

#include <algorithm>
#include <type_traits>

namespace gm {
namespace {

// ------------------------------------------------------------- simple kernels
// Any layout within the bounds: lanes (edge slot, head) over a target's edges, three
// walks (the maxima, the sums, the weights); gradients of rows by a lane a column.

template <typename T, typename R>
__device__ T rel_head_dot(const RelArgs<T, R>& a, const R* qi, const R* kj, const T* phases, int h) {
  T acc = T(0);
  for (int f = 0; f < a.L.F; ++f) {
    const int n = a.L.n[f], an = a.L.a[f];
    if (n == 0) {
      const int at = a.L.off[f] + h * an;
      for (int u = 0; u < an; ++u) acc += row_widen(qi[at + u]) * row_widen(kj[at + u]);
    } else {
      const int at = a.L.off[f] + 2 * h * an;
      T re = T(0), im = T(0);
      for (int u = 0; u < an; ++u) {
        const T q0 = row_widen(qi[at + 2 * u]), q1 = row_widen(qi[at + 2 * u + 1]);
        const T k0 = row_widen(kj[at + 2 * u]), k1 = row_widen(kj[at + 2 * u + 1]);
        re += q0 * k0 + q1 * k1;
        im += q1 * k0 - q0 * k1;
      }
      acc += phases[2 * n - 2] * re + phases[2 * n - 1] * im;
    }
  }
  return acc;
}

// Edge e's score of head h for the target row qi; -inf outside the window.
template <typename T, typename R>
__device__ __forceinline__ T rel_logit(const RelArgs<T, R>& a, const R* qi, int64_t e, int h) {
  const T* rec = a.records + e * 2 * a.L.orders;
  const T bias = rec[1];
  if (bias == neg_inf<T>()) return bias;
  const T learned = a.table[rel_bucket(rec) * a.L.H + h] * T(kRelLog2e);
  return a.scale * rel_head_dot(a, qi, a.k + (int64_t)rel_source(rec) * a.L.D, rec + 2, h) + (bias + learned);
}

// Maximum over lanes h, h + G, ...: as group_sum.
template <typename T>
__device__ __forceinline__ T rel_group_max(T v, int lane, int G, int S) {
  const int s = lane / G, h = lane % G;
  if (s >= S) v = neg_inf<T>();
  for (int step = 1; step < S; step <<= 1) {
    const int from = lane + step * G;
    const T o = __shfl(v, from < kWave ? from : lane, kWave);
    if ((s % (2 * step)) == 0 && s + step < S) v = o > v ? o : v;
  }
  return __shfl(v, h, kWave);
}

template <typename T, typename R>
__global__ __launch_bounds__(256) void relative_forward_simple(RelArgs<T, R> a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = xcd_block(blockIdx.x, gridDim.x) * kWavesPerBlock + (threadIdx.x >> 6);
  if (i >= a.n_targets) return;
  const int H = a.L.H, S = kWave / H, h = lane % H, s = lane / H;
  const int64_t e0 = a.row_ptr[i], e1 = a.row_ptr[i + 1];
  const R* qi = a.q + i * a.L.D;
  T m = neg_inf<T>(), l = T(0);
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) {
      const T lw = rel_logit(a, qi, e, h);
      m = lw > m ? lw : m;
    }
  m = rel_group_max(m, lane, H, S);
  if (m == neg_inf<T>()) m = T(0);  // no edge inside: every weight is zero
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) l += row_exp2(rel_logit(a, qi, e, h) - m);
  l = group_sum(l, lane, H, S);
  const T inv = l == T(0) ? T(0) : T(1) / l;
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) {
      const T lw = rel_logit(a, qi, e, h);
      a.alpha[e * H + h] = lw == neg_inf<T>() ? T(0) : row_exp2(lw - m) * inv;
    }
}

struct RelColumn {
  int n, h, part, pair;  // pair: the column of the pair's real part
};

template <typename T, typename R>
__device__ RelColumn rel_column(const RelArgs<T, R>& a, int c) {
  int f = 0;
  for (int i = 1; i < a.L.F; ++i)
    if (c >= a.L.off[i]) f = i;
  const int dim = a.L.n[f] == 0 ? 1 : 2, local = c - a.L.off[f];
  return {a.L.n[f], local / dim / a.L.a[f], local % dim, c - local % dim};
}

// kTargets: dq of a target's row, from the keys of its edges; else dk of a source's, from the queries of its edges.
template <typename T, typename R, bool kTargets>
__global__ __launch_bounds__(256) void relative_rows_simple(RelArgs<T, R> a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = xcd_block(blockIdx.x, gridDim.x) * kWavesPerBlock + (threadIdx.x >> 6);
  if (row >= (kTargets ? a.n_targets : a.n_sources)) return;
  const int64_t* ptr = kTargets ? a.row_ptr : a.src_ptr;
  const int64_t e0 = ptr[row], e1 = ptr[row + 1];
  for (int c = lane; c < a.L.D; c += kWave) {
    const RelColumn col = rel_column(a, c);
    T acc = T(0);
    for (int64_t at = e0; at < e1; ++at) {
      const T* rec = (kTargets ? a.records : a.records_s) + at * 2 * a.L.orders;
      const int64_t e = kTargets ? at : rel_index(rec + 1);
      const T ds = a.ds[e * a.L.H + col.h];
      if (ds == T(0)) continue;
      const R* other = kTargets ? a.k + (int64_t)rel_source(rec) * a.L.D : a.q + (int64_t)rel_index(rec) * a.L.D;
      if (col.n == 0) {
        acc += ds * row_widen(other[c]);
      } else {
        const T cr = rec[2 * col.n], ci = kTargets ? rec[2 * col.n + 1] : -rec[2 * col.n + 1];
        const T x0 = row_widen(other[col.pair]), x1 = row_widen(other[col.pair + 1]);
        acc += ds * (col.part == 0 ? cr * x0 - ci * x1 : cr * x1 + ci * x0);
      }
    }
    row_narrow(a.gradient_scale * acc, (kTargets ? a.dq : a.dk)[row * a.L.D + c]);
  }
}

// --------------------------------------------------------------------- ds
// T of a target and ds of its edges, which are added to the wave's bins (buckets, columns) in LDS.  Lanes (edge slot,
// head) read alpha and g, which lie edge by edge, as whole lines; a wave holds kRelHeld steps of both, so that a row
// of up to that many (times the waves it is shared by) is read once.  The workgroups are persistent, find their next
// row while the present one's numbers are on their way, and each writes a row of bins.  Bound by bytes and by how many
// are on their way: 63 million edges of eight heads take 1.50 ms, 6.1 GB read and written (4.1 TB/s).
// Holding 16 steps takes as long, 8 takes 5 % more: long rows are read twice.
//
// A bin is a slot's own, added to in the order of its steps, while the bins take up to kRelBins bytes a wave; of more
// buckets several slots share one and add one after the other (a wave's LDS operations are done in order): two of them
// may hold edges of one bucket.  A read, an add and a write, not LDS's atomic add: that takes a cycle a lane (2.9 ms
// against 1.9, before the loads of a row were all requested together).

constexpr int kRelHeld = 12;
constexpr int kRelBins = 8 * 1024;

template <typename T>
struct RelScores {
  int H, S, buckets, shares;  // shares: the slots that add to one bin
  const int64_t* row_ptr;
  const int32_t* order;       // the rows by length, or null: as they come
  uint32_t shared, rows;      // the first `shared` are a workgroup's each, the others a wave's
  const uint8_t* bucket;      // (n_edges)
  const T* alpha;
  const T* g;
  T* ds;
  T* partial;
};

// `count` numbers from p as a buffer: what is read past them is zero, what is written there is dropped.
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rel_span(const T* p, int count) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(p), (short)0, count * (int)sizeof(T), 0x00020000);
}
typedef uint32_t rel_u2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ __forceinline__ T rel_read(__amdgpu_buffer_rsrc_t r, int off) {
  if constexpr (sizeof(T) == 8)
    return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
  else
    return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}
template <typename T>
__device__ __forceinline__ void rel_write(T v, __amdgpu_buffer_rsrc_t r, int off) {
  if constexpr (sizeof(T) == 8)
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(rel_u2, v), r, off, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, v), r, off, 0, 0);
}

template <typename T>
__global__ __launch_bounds__(256) void relative_scores(RelScores<T> a, uint32_t blocks) {
  extern __shared__ __align__(16) char rel_lds[];
  const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6)), H = a.H, S = a.S;
  const int s = lane / H, h = lane % H;
  const bool on = s < S;
  T* shared = reinterpret_cast<T*>(rel_lds);  // (waves, H): a row's waves' parts of T
  T* all = shared + kWavesPerBlock * H;
  const int columns = (S + a.shares - 1) / a.shares * H, size = a.buckets * columns;
  T* bins = all + wave * size;
  T* bin = bins + (on ? s / a.shares * H + h : 0);
  const int turn = s % a.shares;
  const int step = S * H * (int)sizeof(T);                         // a step's bytes
  const int mine = on ? lane * (int)sizeof(T) : (int)0xC0000000u;  // past every span
  for (int i = lane; i < size; i += kWave) bins[i] = T(0);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  // the edges of this wave in a block's row (whole: of the workgroup's); none where the wave has no row
  struct Range {
    int64_t e0, e1;
  };
  auto range = [&](uint32_t block) {
    if (block >= blocks) return Range{0, 0};
    const bool whole = block < a.shared;
    uint32_t at = xcd_spread_block32(whole ? block : block - a.shared, whole ? a.shared : blocks - a.shared);
    if (!whole) at = a.shared + at * kWavesPerBlock + wave;
    if (at >= a.rows) return Range{0, 0};
    const uint32_t row = a.order ? uniform((int)a.order[at]) : at;
    const int64_t r0 = uniform(a.row_ptr[row]), r1 = uniform(a.row_ptr[row + 1]);
    if (!whole) return Range{r0, r1};
    const uint32_t steps = ((uint32_t)(r1 - r0) + S - 1) / S, per = (steps + kWavesPerBlock - 1) / kWavesPerBlock * S;
    const int64_t first = r0 + (int64_t)wave * per, e0 = first < r1 ? first : r1;
    return Range{e0, e0 + per < r1 ? e0 + per : r1};
  };
  Range next = range(blockIdx.x);
  for (uint32_t block = blockIdx.x; block < blocks; block += gridDim.x) {
    const bool whole = block < a.shared;
    const int64_t e0 = next.e0, e1 = next.e1;
    next = range(block + gridDim.x);  // found while this row's numbers are on their way
    T al[kRelHeld], g[kRelHeld];
    int b[kRelHeld];
    // the steps from edge e; what lies past the row's share (and lanes without a head) reads as zero
    auto read = [&](int64_t e) {
      const int left = (int)(e1 - e < kRelHeld * S ? e1 - e : kRelHeld * S);
      const auto al_of = rel_span(a.alpha + e * H, left * H), g_of = rel_span(a.g + e * H, left * H);
      const auto b_of = rel_span(a.bucket + e, left);
#pragma unroll
      for (int n = 0; n < kRelHeld; ++n) {
        al[n] = rel_read<T>(al_of, mine + n * step);
        g[n] = rel_read<T>(g_of, mine + n * step);
        b[n] = __builtin_amdgcn_raw_buffer_load_b8(b_of, s + n * S, 0, 0);
      }
    };
    const bool once = e1 - e0 <= kRelHeld * S;
    T total = T(0);
    for (int64_t e = e0; e < e1; e += kRelHeld * S) {
      read(e);
#pragma unroll
      for (int n = 0; n < kRelHeld; ++n) total += al[n] != T(0) ? al[n] * g[n] : T(0);
    }
    total = group_sum(total, lane, H, S);
    if (whole) {
      __syncthreads();
      if (lane < H) shared[wave * H + lane] = total;
      __syncthreads();
      total = shared[h];
      for (int o = 1; o < kWavesPerBlock; ++o) total += shared[o * H + h];
    }
    for (int64_t e = e0; e < e1; e += kRelHeld * S) {
      if (!once) read(e);
      const int left = (int)(e1 - e < kRelHeld * S ? e1 - e : kRelHeld * S);
      const auto ds_of = rel_span(a.ds + e * H, left * H);
#pragma unroll
      for (int n = 0; n < kRelHeld; ++n) {
        if (n * S < left) {
          const T d = al[n] != T(0) ? al[n] * (g[n] - total) : T(0);
          rel_write(d, ds_of, mine + n * step);
          T* to = bin + b[n] * columns;
          if (a.shares == 1) {
            if (on) *to += d;  // this lane's alone
          } else {
            for (int o = 0; o < a.shares; ++o) {
              if (on && turn == o) *to += d;
              wave_lds();
            }
          }
        }
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.buckets * H; i += blockDim.x) {
    const int bucket = i / H, head = i % H;
    T v = T(0);
    for (int w = 0; w < kWavesPerBlock; ++w)
      for (int c = head; c < columns; c += H) v += all[w * size + bucket * columns + c];
    a.partial[(int64_t)blockIdx.x * a.buckets * H + i] = v;
  }
}

// ------------------------------------------------------------------- repack
// Rows of heads from one layout into another of the same heads with more or fewer copies: what is missing is zero, what
// is over is left out.  A workgroup finds its columns once and takes rows until none is left.

template <typename R>
__global__ __launch_bounds__(256) void relative_repack(HeadsLayout from, HeadsLayout to, const R* src, int64_t n_rows,
                                                       R* dst) {
  __shared__ int place[GM_ATTN_MAX_D];
  for (int c = threadIdx.x; c < to.D; c += blockDim.x) {
    int f = 0;
    for (int i = 1; i < to.F; ++i)
      if (c >= to.off[i]) f = i;
    const int dim = to.n[f] == 0 ? 1 : 2, local = c - to.off[f], h = local / (to.a[f] * dim);
    const int at = local - h * to.a[f] * dim;
    place[c] = -1;
    for (int i = 0; i < from.F; ++i)
      if (from.n[i] == to.n[f] && at < from.a[i] * dim) place[c] = from.off[i] + h * from.a[i] * dim + at;
  }
  __syncthreads();
  for (int64_t row = blockIdx.x; row < n_rows; row += gridDim.x)
    for (int c = threadIdx.x; c < to.D; c += blockDim.x)
      dst[row * to.D + c] = place[c] < 0 ? R(0) : src[row * from.D + place[c]];
}

// ------------------------------------------------------------------- launch

int rel_parse(const int64_t* desc, int64_t F, int64_t H, int64_t D, int64_t orders, RelLayout& L) {
  GM_REQUIRE(orders >= 1 && orders <= 256, "the phase tables need at least one order, 256 at most");
  const int rc = parse_heads(desc, F, H, GM_ATTN_MAX_H, D, L);
  if (rc != GM_OK) return rc;
  L.orders = (int)orders;
  GM_REQUIRE(L.n[L.F - 1] < L.orders, "a descriptor frequency exceeds the phase tables");
  return GM_OK;
}

template <typename T, typename R>
int rel_prepare(RelArgs<T, R>& a, const T* records, const int64_t* desc, const int64_t* row_ptr, int64_t n_targets,
                int64_t n_sources, int64_t n_edges, int64_t D, int64_t orders, int64_t F, int64_t H, int64_t buckets,
                double scale, const R* q, const R* k) {
  GM_REQUIRE(n_targets >= 0 && n_sources >= 0 && n_edges >= 0, "sizes must be non-negative");
  GM_REQUIRE(n_targets < (int64_t(1) << 31) && n_sources < (int64_t(1) << 31) && n_edges < (int64_t(1) << 31),
             "the records index nodes and edges in 32 bits");
  GM_REQUIRE((!std::is_same<T, float>::value) || n_sources <= (int64_t(1) << 24),
             "float records index sources in 24 bits");
  GM_REQUIRE(buckets >= 1 && buckets <= kRelMaxBuckets, "1 to 256 buckets");
  const int rc = rel_parse(desc, F, H, D, orders, a.L);
  if (rc != GM_OK) return rc;
  if (n_targets > 0) GM_REQUIRE(q && row_ptr, "q and row_ptr must be device pointers");
  if (n_edges > 0) GM_REQUIRE(k && records, "k and the records must be device pointers");
  a.buckets = (int)buckets;
  a.q = q;
  a.k = k;
  a.records = records;
  a.row_ptr = row_ptr;
  a.n_targets = n_targets;
  a.n_sources = n_sources;
  a.n_edges = n_edges;
  a.scale = (T)(scale * kRelLog2e);
  a.gradient_scale = (T)scale;
  a.by_heads = 65536u / (uint32_t)H + 1;
  return GM_OK;
}

// The rows' classes; order null: none.
int rel_rows(const int32_t* order, const int64_t* counts, int64_t n, RelRows& rows) {
  rows = RelRows{order, {0, 0, 0}};
  if (!order) return GM_OK;
  GM_REQUIRE(counts, "the classes' counts (a host array of three) are required");
  int64_t sum = 0;
  for (int c = 0; c < 3; ++c) {
    GM_REQUIRE(counts[c] >= 0, "a class has a negative count");
    rows.count[c] = counts[c];
    sum += counts[c];
  }
  GM_REQUIRE(sum == n, "the classes must hold every row once");
  return GM_OK;
}

// Whether the lane kernels can run: they serve the layout, and the addresses are whole.
template <typename T, typename R>
int rel_lanes_check(const RelArgs<T, R>& a) {
  GM_REQUIRE((std::is_same<T, float>::value) && rel_slots(a.L) > 0, "the lane kernels do not serve this layout");
  GM_REQUIRE(aligned(a.q, 16) && aligned(a.k, 16) && aligned(a.dq, 16) && aligned(a.dk, 16) &&
                 aligned(a.records, 8) && aligned(a.pairs, 8) && aligned(a.pairs_s, 8),
             "the lane kernels take rows at multiples of 16 bytes, records and entries of 8");
  return GM_OK;
}

template <typename T, typename R>
int relative_forward(const R* q, const R* k, const T* table, const T* records, const int64_t* desc,
                     const int64_t* row_ptr, const int32_t* order, const int64_t* counts, int64_t n_targets,
                     int64_t n_sources, int64_t n_edges, int64_t D, int64_t orders, int64_t F, int64_t H,
                     int64_t buckets, double scale, T* alpha, void* stream) {
  RelArgs<T, R> a{};
  const int rc = rel_prepare(a, records, desc, row_ptr, n_targets, n_sources, n_edges, D, orders, F, H, buckets, scale,
                             q, k);
  if (rc != GM_OK) return rc;
  if (n_targets == 0 || n_edges == 0) return GM_OK;
  GM_REQUIRE(alpha && table, "alpha and table must be device pointers");
  a.alpha = alpha;
  a.table = table;
  if constexpr (std::is_same<T, float>::value) {
    if (order) {
      RelRows rows;
      int status = rel_lanes_check(a);
      if (status == GM_OK) status = rel_rows(order, counts, n_targets, rows);
      return status == GM_OK ? rel_launch_units(RelPass::Forward, a, rows, (hipStream_t)stream) : status;
    }
  }
  GM_REQUIRE(!order, "the lane kernels take float tables");
  hipLaunchKernelGGL((relative_forward_simple<T, R>), dim3((unsigned)blocks_for(n_targets)), dim3(256), 0,
                     (hipStream_t)stream, a);
  return check_launch("relative_forward");
}

// ds of every edge, and the sums of its buckets.
template <typename T, typename R>
int relative_scores_launch(const RelArgs<T, R>& a, const RelRows& rows, const uint8_t* bucket, T* dtable,
                           hipStream_t stream) {
  RelScores<T> k{};
  k.H = a.L.H;
  k.S = kWave / a.L.H;
  k.buckets = a.buckets;
  for (k.shares = 1; k.shares < k.S; k.shares *= 2)
    if ((size_t)a.buckets * ((k.S + k.shares - 1) / k.shares) * a.L.H * sizeof(T) <= kRelBins) break;
  k.shares = std::min(k.shares, k.S);
  k.row_ptr = a.row_ptr;
  k.order = rows.order;
  k.shared = rows.order ? (uint32_t)(rows.count[0] + rows.count[1]) : 0;
  k.rows = (uint32_t)a.n_targets;
  k.bucket = bucket;
  k.alpha = a.alpha;
  k.g = a.g;
  k.ds = a.ds;
  k.partial = a.partial;
  const int columns = (k.S + k.shares - 1) / k.shares * a.L.H;
  const size_t lds = sizeof(T) * kWavesPerBlock * ((size_t)a.L.H + (size_t)a.buckets * columns);
  const auto kernel = &relative_scores<T>;
  if (lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess)
    return check_launch("relative (LDS)");
  const int64_t blocks = k.shared + blocks_for(a.n_targets - k.shared);
  const int64_t resident = resident_blocks(reinterpret_cast<const void*>(kernel), 256, lds);
  const int64_t most = std::min<int64_t>(kRelTableRows, resident > 0 ? resident : blocks);
  const int64_t grid = std::max<int64_t>(1, std::min(blocks, most));
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), lds, stream, k, (uint32_t)blocks);
  launch_partial_sum<T>(a.partial, grid, a.buckets * a.L.H, dtable, stream);
  return check_launch("relative_scores");
}

template <typename T, typename R>
int relative_backward(const T* g, const T* alpha, const R* q, const R* k, const T* records, const T* records_s,
                      const uint8_t* bucket, const int64_t* desc, const int64_t* row_ptr, const int64_t* src_ptr,
                      const int32_t* order, const int64_t* counts, const float* pairs, const int64_t* pair_ptr,
                      const int32_t* pair_order, const int64_t* pair_counts, const float* pairs_s,
                      const int64_t* pair_ptr_s, const int32_t* pair_order_s, const int64_t* pair_counts_s,
                      int64_t n_targets, int64_t n_sources, int64_t n_edges, int64_t D, int64_t orders, int64_t F,
                      int64_t H, int64_t buckets, double scale, T* ds, T* partial, R* dq, R* dk, T* dtable,
                      void* stream) {
  RelArgs<T, R> a{};
  const int rc = rel_prepare(a, records, desc, row_ptr, n_targets, n_sources, n_edges, D, orders, F, H, buckets, scale,
                             q, k);
  if (rc != GM_OK) return rc;
  GM_REQUIRE(partial && dtable, "partial and dtable must be device pointers");
  if (n_targets > 0) GM_REQUIRE(dq, "dq must be a device pointer");
  if (n_sources > 0) GM_REQUIRE(dk, "dk must be a device pointer");
  const bool lanes = pairs && pairs_s;
  GM_REQUIRE(!pairs == !pairs_s, "both sides' pairs, or neither's");
  if (n_edges > 0) GM_REQUIRE(g && alpha && ds && bucket, "g, alpha, ds and the buckets must be device pointers");
  if (n_edges > 0 && !lanes) GM_REQUIRE(records_s, "the sources' records must be a device pointer");
  if (n_sources > 0 && !lanes) GM_REQUIRE(src_ptr, "src_ptr must be a device pointer");
  a.g = g;
  a.alpha = const_cast<T*>(alpha);  // read only here
  a.records_s = records_s;
  a.src_ptr = src_ptr;
  a.ds = ds;
  a.partial = partial;
  a.dq = dq;
  a.dk = dk;
  const hipStream_t s = (hipStream_t)stream;
  RelRows targets;
  int status = rel_rows(order, counts, n_targets, targets);
  if (status != GM_OK) return status;
  if constexpr (std::is_same<T, float>::value) {
    if (lanes) {
      if (n_targets > 0) GM_REQUIRE(pair_ptr && pair_order, "the pairs' offsets and classes must be device pointers");
      if (n_sources > 0)
        GM_REQUIRE(pair_ptr_s && pair_order_s, "the pairs' offsets and classes must be device pointers");
      a.pairs = pairs;
      a.pair_ptr = pair_ptr;
      a.pairs_s = pairs_s;
      a.pair_ptr_s = pair_ptr_s;
      RelRows rows, rows_s;
      status = rel_lanes_check(a);
      if (status == GM_OK) status = rel_rows(pair_order, pair_counts, (n_targets + 1) / 2, rows);
      if (status == GM_OK) status = rel_rows(pair_order_s, pair_counts_s, (n_sources + 1) / 2, rows_s);
      if (status == GM_OK) status = relative_scores_launch(a, targets, bucket, dtable, s);
      if (status == GM_OK) status = rel_launch_units(RelPass::BackwardTarget, a, rows, s);
      return status == GM_OK ? rel_launch_units(RelPass::BackwardSource, a, rows_s, s) : status;
    }
  }
  GM_REQUIRE(!lanes, "the lane kernels take float tables");
  status = relative_scores_launch(a, targets, bucket, dtable, s);
  if (status != GM_OK) return status;
  if (n_targets > 0)
    hipLaunchKernelGGL((relative_rows_simple<T, R, true>), dim3((unsigned)blocks_for(n_targets)), dim3(256), 0, s, a);
  if (n_sources > 0)
    hipLaunchKernelGGL((relative_rows_simple<T, R, false>), dim3((unsigned)blocks_for(n_sources)), dim3(256), 0, s, a);
  return check_launch("relative_backward");
}

template <typename R>
int relative_repack_rows(const R* src, const int64_t* desc, int64_t F, int64_t D, const int64_t* to_desc, int64_t to_F,
                         int64_t to_D, int64_t H, int64_t n_rows, R* dst, void* stream) {
  HeadsLayout from, to;
  int rc = parse_heads(desc, F, H, GM_ATTN_MAX_H, D, from);
  if (rc == GM_OK) rc = parse_heads(to_desc, to_F, H, GM_ATTN_MAX_H, to_D, to);
  if (rc != GM_OK) return rc;
  GM_REQUIRE(n_rows >= 0, "sizes must be non-negative");
  if (n_rows == 0) return GM_OK;
  GM_REQUIRE(src && dst, "src and dst must be device pointers");
  hipLaunchKernelGGL(relative_repack<R>, dim3((unsigned)std::min<int64_t>(n_rows, 4096)), dim3(256), 0,
                     (hipStream_t)stream, from, to, src, n_rows, dst);
  return check_launch("relative_repack");
}

}  // namespace
}  // namespace gm

extern "C" int gm_relative_padded(const int64_t* desc, int64_t F, int64_t H, int64_t D, int64_t orders,
                                  int64_t* copies) {
  GM_REQUIRE(copies, "copies must be a host array of three");
  gm::RelLayout L{};
  const int rc = gm::rel_parse(desc, F, H, D, orders, L);
  if (rc != GM_OK) return rc;
  int found[3] = {0, 0, 0};
  (void)gm::rel_padded(L, found);
  for (int n = 0; n < 3; ++n) copies[n] = found[n];
  return GM_OK;
}

extern "C" int gm_relative_repack_f32(const float* src, const int64_t* desc, int64_t F, int64_t D,
                                      const int64_t* to_desc, int64_t to_F, int64_t to_D, int64_t H, int64_t n_rows,
                                      float* dst, void* stream) {
  return gm::relative_repack_rows(src, desc, F, D, to_desc, to_F, to_D, H, n_rows, dst, stream);
}
extern "C" int gm_relative_repack_bf16(const uint16_t* src, const int64_t* desc, int64_t F, int64_t D,
                                       const int64_t* to_desc, int64_t to_F, int64_t to_D, int64_t H, int64_t n_rows,
                                       uint16_t* dst, void* stream) {
  return gm::relative_repack_rows(src, desc, F, D, to_desc, to_F, to_D, H, n_rows, dst, stream);
}

extern "C" int64_t gm_relative_partial_rows(void) { return gm::kRelTableRows; }

extern "C" int gm_relative_slots(const int64_t* desc, int64_t F, int64_t H, int64_t D, int64_t orders,
                                 int64_t* slots) {
  GM_REQUIRE(slots, "slots must be a host pointer");
  gm::RelLayout L{};
  const int rc = gm::rel_parse(desc, F, H, D, orders, L);
  if (rc != GM_OK) return rc;
  *slots = gm::rel_slots(L);
  return GM_OK;
}

// T: the arithmetic's type, R the rows'.
#define GM_RELATIVE_ENTRY(SFX, T, R)                                                                                  \
  extern "C" int gm_relative_forward_##SFX(                                                                           \
      const R* q, const R* k, const T* table, const T* records, const int64_t* desc, const int64_t* row_ptr,          \
      const int32_t* order, const int64_t* counts, int64_t n_targets, int64_t n_sources, int64_t n_edges, int64_t D,  \
      int64_t orders, int64_t F, int64_t H, int64_t buckets, double scale, T* alpha, void* stream) {                  \
    return gm::relative_forward<T, R>(q, k, table, records, desc, row_ptr, order, counts, n_targets, n_sources,       \
                                      n_edges, D, orders, F, H, buckets, scale, alpha, stream);                       \
  }                                                                                                                   \
  extern "C" int gm_relative_backward_##SFX(                                                                          \
      const T* g, const T* alpha, const R* q, const R* k, const T* records, const T* records_s,                       \
      const uint8_t* bucket, const int64_t* desc, const int64_t* row_ptr, const int64_t* src_ptr,                     \
      const int32_t* order, const int64_t* counts, const float* pairs, const int64_t* pair_ptr,                       \
      const int32_t* pair_order, const int64_t* pair_counts, const float* pairs_s, const int64_t* pair_ptr_s,         \
      const int32_t* pair_order_s, const int64_t* pair_counts_s, int64_t n_targets, int64_t n_sources,                \
      int64_t n_edges, int64_t D, int64_t orders, int64_t F, int64_t H, int64_t buckets, double scale, T* ds,         \
      T* partial, R* dq, R* dk, T* dtable, void* stream) {                                                            \
    return gm::relative_backward<T, R>(g, alpha, q, k, records, records_s, bucket, desc, row_ptr, src_ptr, order,     \
                                       counts, pairs, pair_ptr, pair_order, pair_counts, pairs_s, pair_ptr_s,         \
                                       pair_order_s, pair_counts_s, n_targets, n_sources, n_edges, D, orders, F, H,   \
                                       buckets, scale, ds, partial, dq, dk, dtable, stream);                          \
  }

GM_RELATIVE_ENTRY(f32, float, float)
GM_RELATIVE_ENTRY(f64, double, double)
GM_RELATIVE_ENTRY(bf16, float, uint16_t)
