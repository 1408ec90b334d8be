// The neighbourhood softmax with a learned relative bias over CSR neighbour lists,
// forward and backward.  Per edge e = (i <- j) in bucket b(e) and head h:
//   s_h   = scale sum_n Re< q_i,n,h , tau_n(e) k_j,n,h > + bias(e) + table[b(e), h]
//   alpha = softmax of s_h over i's edges inside the window (zero outside; a target
//           with no edge inside has only zeros)
// and from g = d alpha, with T_h(i) = sum_e alpha g:
//   ds = alpha (g - T),   dtable[b, h] = sum of ds over the edges of bucket b
//   dq_i = scale sum_e ds tau k_j,   dk_j = scale sum_e ds conj(tau) q_i
//
// The backward reads the forward's weights: a score is formed once.  The pass over
// the targets walks alpha and g, which lie edge by edge, for T, then writes ds and
// adds dq and the buckets' sums; the pass over the sources reads ds.  An edge of
// weight zero counts for nothing, whatever its rows and its g hold: so do the edges
// outside the window.  No atomics between waves: sums are in a fixed order.
//
// Per edge a pass reads one record of 32-bit words (64-bit for double): the source
// with the bucket above it, the bias in units of log 2 (-inf outside the window) and
// the transport's (cos, sin) of orders 1 .., packed once for an edge set; the source
// side's name the target and the edge.
#include "relative.hpp"
#include "partial_sum.hpp"

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

// T of a target and ds of its edges.
template <typename T, typename R>
__global__ __launch_bounds__(256) void relative_scores_simple(RelArgs<T, R> a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = xcd_block(blockIdx.x, gridDim.x) * kWavesPerBlock + (threadIdx.x >> 6);
  if (i >= a.n_targets) return;
  const int H = a.L.H, S = kWave / H, h = lane % H, s = lane / H;
  const int64_t e0 = a.row_ptr[i], e1 = a.row_ptr[i + 1];
  T total = T(0);
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) {
      const T w = a.alpha[e * H + h];
      if (w != T(0)) total += w * a.g[e * H + h];
    }
  total = group_sum(total, lane, H, S);
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) {
      const T w = a.alpha[e * H + h];
      a.ds[e * H + h] = w != T(0) ? w * (a.g[e * H + h] - total) : T(0);
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

// ------------------------------------------------------------------- dtable
// A wave a workgroup over a range of the edges, its bins (buckets, H) in LDS.  The edge
// slots of a step add one after the other: two may hold edges of one bucket, and a
// wave's LDS operations are done in order.  Then the rows of bins are added in double.

template <typename T, typename R>
__global__ __launch_bounds__(64) void relative_table_simple(RelArgs<T, R> a) {
  extern __shared__ __align__(16) char rel_lds[];
  T* bins = reinterpret_cast<T*>(rel_lds);
  const int lane = threadIdx.x, H = a.L.H, S = kWave / H, h = lane % H, s = lane / H;
  for (int i = lane; i < a.buckets * H; i += kWave) bins[i] = T(0);
  __syncthreads();
  const int64_t per = ((a.n_edges + gridDim.x - 1) / gridDim.x + S - 1) / S * S;
  const int64_t e0 = (int64_t)blockIdx.x * per, e1 = e0 + per < a.n_edges ? e0 + per : a.n_edges;
  for (int64_t e = e0; e < e1; e += S) {
    const bool live = s < S && e + s < e1;
    const T v = live ? a.ds[(e + s) * H + h] : T(0);
    const int at = live ? rel_bucket(a.records + (e + s) * 2 * a.L.orders) * H + h : 0;
    for (int t = 0; t < S; ++t) {
      if (s == t && live) bins[at] += v;
      __syncthreads();  // one wave: its LDS reads after its writes
    }
  }
  for (int i = lane; i < a.buckets * H; i += kWave) a.partial[(int64_t)blockIdx.x * a.buckets * H + i] = bins[i];
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
  return GM_OK;
}

// The rows' classes (order null: the simple kernels), which the lane kernels must serve.
template <typename T, typename R>
int rel_rows(const RelArgs<T, R>& a, const int32_t* order, const int64_t* counts, int64_t n, RelRows& rows) {
  rows = RelRows{order, {0, 0, 0}};
  if (!order) return GM_OK;
  GM_REQUIRE((std::is_same<T, float>::value) && rel_slots(a.L) > 0, "the lane kernels do not serve this layout");
  GM_REQUIRE(counts, "the classes' counts (a host array of three) are required");
  int64_t sum = 0;
  for (int c = 0; c < 3; ++c) {
    GM_REQUIRE(counts[c] >= 0, "a class has a negative count");
    rows.count[c] = counts[c];
    sum += counts[c];
  }
  GM_REQUIRE(sum == n, "the classes must hold every row once");
  GM_REQUIRE(aligned(a.q, 16) && aligned(a.k, 16) && aligned(a.dq, 16) && aligned(a.dk, 16) && aligned(a.records, 8) &&
                 aligned(a.records_s, 8),
             "the lane kernels take rows at multiples of 16 bytes, records of 8");
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
  RelRows rows;
  const int status = rel_rows(a, order, counts, n_targets, rows);
  if (status != GM_OK) return status;
  if constexpr (std::is_same<T, float>::value) {
    if (order) return rel_launch_units(RelPass::Forward, a, rows, (hipStream_t)stream);
  }
  hipLaunchKernelGGL((relative_forward_simple<T, R>), dim3((unsigned)blocks_for(n_targets)), dim3(256), 0,
                     (hipStream_t)stream, a);
  return check_launch("relative_forward");
}

template <typename T, typename R>
int relative_backward(const T* g, const T* alpha, const R* q, const R* k, const T* records, const T* records_s,
                      const int64_t* desc, const int64_t* row_ptr, const int64_t* src_ptr, const int32_t* order,
                      const int64_t* counts, const int32_t* order_s, const int64_t* counts_s, int64_t n_targets,
                      int64_t n_sources, int64_t n_edges, int64_t D, int64_t orders, int64_t F, int64_t H,
                      int64_t buckets, double scale, T* ds, T* partial, R* dq, R* dk, T* dtable, void* stream) {
  RelArgs<T, R> a{};
  const int rc = rel_prepare(a, records, desc, row_ptr, n_targets, n_sources, n_edges, D, orders, F, H, buckets, scale,
                             q, k);
  if (rc != GM_OK) return rc;
  GM_REQUIRE(partial && dtable, "partial and dtable must be device pointers");
  if (n_targets > 0) GM_REQUIRE(dq, "dq must be a device pointer");
  if (n_sources > 0) GM_REQUIRE(src_ptr && dk, "src_ptr and dk must be device pointers");
  if (n_edges > 0) GM_REQUIRE(g && alpha && ds && records_s, "g, alpha, ds and the sources' records must be device pointers");
  a.g = g;
  a.alpha = const_cast<T*>(alpha);  // read only here
  a.records_s = records_s;
  a.src_ptr = src_ptr;
  a.ds = ds;
  a.partial = partial;
  a.dq = dq;
  a.dk = dk;
  const hipStream_t s = (hipStream_t)stream;
  const int columns = a.buckets * a.L.H;
  GM_REQUIRE(!order == !order_s || n_targets == 0 || n_sources == 0, "both sides' rows are in classes, or neither's");
  RelRows targets, sources;
  int status = rel_rows(a, order, counts, n_targets, targets);
  if (status == GM_OK) status = rel_rows(a, order_s, counts_s, n_sources, sources);
  if (status != GM_OK) return status;
  if constexpr (std::is_same<T, float>::value) {
    if (order || order_s) {
      status = rel_launch_units(RelPass::BackwardTarget, a, targets, s);
      if (status == GM_OK) status = rel_launch_units(RelPass::BackwardSource, a, sources, s);
      if (status != GM_OK) return status;
      launch_partial_sum<T>(partial, kRelTableRows, columns, dtable, s);
      return check_launch("relative_backward");
    }
  }
  if (n_targets > 0) {
    const dim3 grid((unsigned)blocks_for(n_targets));
    hipLaunchKernelGGL((relative_scores_simple<T, R>), grid, dim3(256), 0, s, a);
    hipLaunchKernelGGL((relative_rows_simple<T, R, true>), grid, dim3(256), 0, s, a);
  }
  if (n_sources > 0)
    hipLaunchKernelGGL((relative_rows_simple<T, R, false>), dim3((unsigned)blocks_for(n_sources)), dim3(256), 0, s, a);
  hipLaunchKernelGGL((relative_table_simple<T, R>), dim3(kRelTableRows), dim3(kWave), sizeof(T) * columns, s, a);
  launch_partial_sum<T>(partial, kRelTableRows, columns, dtable, s);
  return check_launch("relative_backward");
}

}  // namespace
}  // namespace gm

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
      const T* g, const T* alpha, const R* q, const R* k, const T* records, const T* records_s, const int64_t* desc,  \
      const int64_t* row_ptr, const int64_t* src_ptr, const int32_t* order, const int64_t* counts,                    \
      const int32_t* order_s, const int64_t* counts_s, int64_t n_targets, int64_t n_sources, int64_t n_edges,         \
      int64_t D, int64_t orders, int64_t F, int64_t H, int64_t buckets, double scale, T* ds, T* partial, R* dq,       \
      R* dk, T* dtable, void* stream) {                                                                               \
    return gm::relative_backward<T, R>(g, alpha, q, k, records, records_s, desc, row_ptr, src_ptr, order, counts,     \
                                       order_s, counts_s, n_targets, n_sources, n_edges, D, orders, F, H, buckets,    \
                                       scale, ds, partial, dq, dk, dtable, stream);                                   \
  }

GM_RELATIVE_ENTRY(f32, float, float)
GM_RELATIVE_ENTRY(f64, double, double)
GM_RELATIVE_ENTRY(bf16, float, uint16_t)
