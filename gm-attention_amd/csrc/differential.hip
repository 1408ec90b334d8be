// The differential neighbourhood softmax over CSR neighbour lists, forward and
// backward.  Head h has two score maps p = 2 h, 2 h + 1; the rows of q and k are
// the direct sum of the 2 H maps, map-major within each frequency.  Per edge
// e = (i <- j):
//   s_p = scale sum_n Re< q_i,n,p , tau_n(e) k_j,n,p > + bias(e)
//   a_p = softmax of s_p over i's edges inside the window (zero outside; a target
//         with no edge inside has only zeros)
//   alpha_h = a_2h - lambda_h a_2h+1
// and from g = d alpha, with c_2h = 1, c_2h+1 = -lambda_h, T_p(i) = sum_e a_p g_h:
//   ds_p = scale c_p a_p (g_h - T_p)
//   dq_i = sum_e ds tau k_j,  dk_j = sum_e ds conj(tau) q_i
//   dlambda_h = - sum_i T_2h+1(i).
//
// Neither the maps nor ds are written: the forward keeps the maximum of s_p and its
// weights' sum for every target, the backward forms a_p again from them.  The pass over the targets needs
// no second walk for T either: sum ds tau k = scale c (sum a g tau k - T sum a tau k),
// two sums beside T in one walk.  What a row's g share cancels in that difference and
// leaves the roundings of both sums, where a second walk over a (g - T) would leave
// T's: twice as far off for g = 10 + N(0, 1) over 120 edges (3.3e-6 against 1.7e-6 of
// the result in float32), nothing without a common part (2.4e-7 against 2.1e-7).  The
// pass over the sources reads T and both numbers of its edges' targets.  No atomics:
// sums are in a fixed order.
//
// Per edge both passes read one record of 32-bit words (64-bit for double): the
// other node, the bias (in units of log 2, as the scores here; -inf outside the
// window) and the transport's (cos, sin) of orders 1 .., packed once for an edge
// set; the source side's, in the order of the edges sorted by source, name the edge
// too, whose g they read.
#include "differential.hpp"

namespace gm {
namespace {

template <typename T>
struct DfWord {
  using type = int32_t;
};
template <>
struct DfWord<double> {
  using type = int64_t;
};

template <typename T>
__device__ __forceinline__ int64_t node_of(const T* word) {
  return *reinterpret_cast<const typename DfWord<T>::type*>(word);
}

// ------------------------------------------------------------- generic path
// Any layout within the bounds: lanes (edge slot, map) over a target's edges, three
// walks (the maxima, the sums, the weights); gradients of rows by a lane a column.

template <typename T, typename R>
__device__ T generic_map_score(const DfArgs<T, R>& a, const R* qi, const R* kj, const T* phases, int p) {
  T acc = T(0);
  for (int f = 0; f < a.L.F; ++f) {
    const int n = a.L.n[f], an = a.L.a[f];
    if (n == 0) {
      const int at = a.L.off[f] + p * an;
      for (int u = 0; u < an; ++u) acc += row_widen(qi[at + u]) * row_widen(kj[at + u]);
    } else {
      const int at = a.L.off[f] + 2 * p * an;
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

// Edge e's score of map p for the target row qi; -inf outside the window.
template <typename T, typename R>
__device__ __forceinline__ T generic_logit(const DfArgs<T, R>& a, const R* qi, int64_t e, int p) {
  const T* rec = a.records + e * 2 * a.L.orders;
  const T bias = rec[1];
  if (bias == neg_inf<T>()) return bias;
  return a.scale * generic_map_score(a, qi, a.k + node_of(rec) * a.L.D, rec + 2, p) + bias;
}

// Maximum over lanes h, h + G, ...: as group_sum.
template <typename T>
__device__ __forceinline__ T group_max(T v, int lane, int G, int S) {
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
__global__ __launch_bounds__(256) void differential_forward_generic(DfArgs<T, R> a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = xcd_block(blockIdx.x, gridDim.x) * kWavesPerBlock + (threadIdx.x >> 6);
  if (i >= a.n_targets) return;
  const int P = a.L.P, S = kWave / P, p = lane % P, s = lane / P;
  const int64_t e0 = a.row_ptr[i], e1 = a.row_ptr[i + 1];
  const R* qi = a.q + i * a.L.D;
  T m = neg_inf<T>(), l = T(0);
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) {
      const T lw = generic_logit(a, qi, e, p);
      m = lw > m ? lw : m;
    }
  m = group_max(m, lane, P, S);
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) {
      const T lw = generic_logit(a, qi, e, p);
      if (lw != neg_inf<T>()) l += row_exp2(lw - m);
    }
  l = group_sum(l, lane, P, S);
  const T inv = l == T(0) ? T(0) : T(1) / l;
  if (a.stats && lane < P) {
    a.stats[(i * P + p) * 2] = m == neg_inf<T>() ? T(0) : m;
    a.stats[(i * P + p) * 2 + 1] = inv;
  }
  const T lambda = a.lambda[p >> 1];
  for (int64_t e = e0; e < e1; e += S) {  // whole waves: the pair's second map comes by a shuffle
    const bool live = s < S && e + s < e1;
    T w = T(0);
    if (live) {
      const T lw = generic_logit(a, qi, e + s, p);
      if (lw != neg_inf<T>()) w = row_exp2(lw - m) * inv;
    }
    const T other = __shfl(w, lane | 1, kWave);
    if (live && (p & 1) == 0) a.alpha[(e + s) * a.L.H + (p >> 1)] = w - lambda * other;
  }
}

// T_p of a target and ds of its edges.
template <typename T, typename R>
__global__ __launch_bounds__(256) void differential_backward_scores_generic(DfArgs<T, R> a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = xcd_block(blockIdx.x, gridDim.x) * kWavesPerBlock + (threadIdx.x >> 6);
  if (i >= a.n_targets) return;
  const int P = a.L.P, S = kWave / P, p = lane % P, s = lane / P;
  const int64_t e0 = a.row_ptr[i], e1 = a.row_ptr[i + 1];
  const R* qi = a.q + i * a.L.D;
  const T m = a.stats[(i * P + p) * 2], inv = a.stats[(i * P + p) * 2 + 1];
  T total = T(0);
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) {
      const T lw = generic_logit(a, qi, e, p);
      const T w = lw == neg_inf<T>() ? T(0) : row_exp2(lw - m) * inv;
      if (lw != neg_inf<T>()) total += w * a.g[e * a.L.H + (p >> 1)];
      a.ds[e * P + p] = w;
    }
  total = group_sum(total, lane, P, S);
  if (lane < P) {
    a.rows[(i * P + p) * 3] = m;
    a.rows[(i * P + p) * 3 + 1] = inv;
    a.rows[(i * P + p) * 3 + 2] = total;
  }
  const T factor = a.gradient_scale * ((p & 1) ? -a.lambda[p >> 1] : T(1));
  if (s < S)
    for (int64_t e = e0 + s; e < e1; e += S) {
      const T w = a.ds[e * P + p];
      const bool in = a.records[e * 2 * a.L.orders + 1] != neg_inf<T>();
      a.ds[e * P + p] = in ? factor * w * (a.g[e * a.L.H + (p >> 1)] - total) : T(0);
    }
}

struct DfColumn {
  int n, p, part, pair;  // pair: the column of the pair's real part; p < 0: no map's column
};

template <typename T, typename R>
__device__ DfColumn locate_column(const DfArgs<T, R>& a, int c) {
  for (int f = 0; f < a.L.F; ++f) {
    const int dim = a.L.n[f] == 0 ? 1 : 2, local = c - a.L.off[f];
    if (local >= 0 && local < a.L.P * a.L.a[f] * dim)
      return {a.L.n[f], local / dim / a.L.a[f], local % dim, c - local % dim};
  }
  return {0, -1, 0, c};
}

template <typename T, typename R>
__global__ __launch_bounds__(256) void differential_backward_target_generic(DfArgs<T, R> a) {
  const int lane = threadIdx.x & 63;
  const int64_t i = xcd_block(blockIdx.x, gridDim.x) * kWavesPerBlock + (threadIdx.x >> 6);
  if (i >= a.n_targets) return;
  const int64_t e0 = a.row_ptr[i], e1 = a.row_ptr[i + 1];
  for (int c = lane; c < a.L.D; c += kWave) {
    const DfColumn col = locate_column(a, c);
    T acc = T(0);
    if (col.p >= 0) {
      for (int64_t e = e0; e < e1; ++e) {
        const T* rec = a.records + e * 2 * a.L.orders;
        if (rec[1] == neg_inf<T>()) continue;
        const T ds = a.ds[e * a.L.P + col.p];
        const R* kj = a.k + node_of(rec) * a.L.D;
        if (col.n == 0) {
          acc += ds * row_widen(kj[c]);
        } else {
          const T cr = rec[2 * col.n], ci = rec[2 * col.n + 1];
          const T k0 = row_widen(kj[col.pair]), k1 = row_widen(kj[col.pair + 1]);
          acc += ds * (col.part == 0 ? cr * k0 - ci * k1 : cr * k1 + ci * k0);
        }
      }
    }
    row_narrow(acc, a.dq[i * a.L.D + c]);
  }
}

template <typename T, typename R>
__global__ __launch_bounds__(256) void differential_backward_source_generic(DfArgs<T, R> a) {
  const int lane = threadIdx.x & 63;
  const int64_t j = xcd_block(blockIdx.x, gridDim.x) * kWavesPerBlock + (threadIdx.x >> 6);
  if (j >= a.n_sources) return;
  const int64_t g0 = a.src_ptr[j], g1 = a.src_ptr[j + 1];
  for (int c = lane; c < a.L.D; c += kWave) {
    const DfColumn col = locate_column(a, c);
    T acc = T(0);
    if (col.p >= 0) {
      for (int64_t g = g0; g < g1; ++g) {
        const T* rec = a.records_s + g * (2 * a.L.orders + 2);
        if (rec[2] == neg_inf<T>()) continue;
        const T ds = a.ds[node_of(rec + 1) * a.L.P + col.p];
        const R* qi = a.q + node_of(rec) * a.L.D;
        if (col.n == 0) {
          acc += ds * row_widen(qi[c]);
        } else {
          const T cr = rec[2 * col.n + 2], ci = rec[2 * col.n + 3];
          const T q0 = row_widen(qi[col.pair]), q1 = row_widen(qi[col.pair + 1]);
          acc += ds * (col.part == 0 ? cr * q0 + ci * q1 : cr * q1 - ci * q0);
        }
      }
    }
    row_narrow(acc, a.dk[j * a.L.D + c]);
  }
}

// ------------------------------------------------------------------ dlambda
// -sum over targets of T of every head's second map, in double, in a fixed order:
// kLambdaBlocks workgroups of a share of the targets each, then one.

constexpr int kLambdaBlocks = 256;

template <typename T>
__global__ __launch_bounds__(256) void differential_lambda_partial(const T* rows, int64_t n_targets, int H,
                                                                   double* partial) {
  __shared__ double sums[256];
  const int per = 256 / H, h = threadIdx.x % H, at = threadIdx.x / H;  // 256 / H targets a step
  double s = 0.0;
  if (at < per)
    for (int64_t i = (int64_t)blockIdx.x * per + at; i < n_targets; i += (int64_t)gridDim.x * per)
      s -= (double)rows[((i * H + h) * 2 + 1) * 3 + 2];
  sums[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < H) {
    double t = 0.0;
    for (int w = 0; w < per; ++w) t += sums[w * H + threadIdx.x];
    partial[(int64_t)blockIdx.x * H + threadIdx.x] = t;
  }
}

template <typename T>
__global__ __launch_bounds__(64) void differential_lambda_sum(const double* partial, int blocks, int H, T* out) {
  double s = 0.0;
  for (int b = threadIdx.x; b < blocks; b += 64) s += partial[(int64_t)b * H + blockIdx.x];
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, kWave);
  if (threadIdx.x == 0) out[blockIdx.x] = (T)s;
}

// ------------------------------------------------------------------- launch

int parse_maps(const int64_t* desc, int64_t F, int64_t H, int64_t D, int64_t orders, DfLayout& L) {
  GM_REQUIRE(desc != nullptr, "desc must be a host pointer to (F, 5) int64");
  GM_REQUIRE(F >= 1 && F <= kDfMaxFreq, "desc must have 1 to 8 frequency rows");
  GM_REQUIRE(H >= 1 && H <= GM_ATTN_MAX_H, "at most 16 heads");
  GM_REQUIRE(D >= 1 && D <= GM_ATTN_MAX_D, "D must be in [1, 1024]");
  GM_REQUIRE(orders >= 1, "the phase tables need at least one order");
  L.F = (int)F;
  L.H = (int)H;
  L.P = 2 * (int)H;
  L.D = (int)D;
  L.orders = (int)orders;
  int64_t next = 0;
  for (int f = 0; f < F; ++f) {
    const int64_t* row = desc + f * GM_ATTN_DESC;
    GM_REQUIRE(row[0] >= 0 && row[0] < orders, "a descriptor frequency exceeds the phase tables");
    GM_REQUIRE(f == 0 || row[0] > desc[(f - 1) * GM_ATTN_DESC], "the descriptor's frequencies must rise");
    GM_REQUIRE(row[4] == (row[0] == 0 ? 1 : 2), "descriptor dim must be 1 at frequency 0 and 2 above");
    GM_REQUIRE(row[1] >= 1 && row[1] <= GM_ATTN_MAX_D && row[2] == next,
               "the descriptor's rows must hold copies and follow each other");
    next += 2 * H * row[1] * row[4];
    GM_REQUIRE(next <= D, "a descriptor row runs past the flat width D");
    L.n[f] = (int)row[0];
    L.a[f] = (int)row[1];
    L.off[f] = (int)row[2];
  }
  GM_REQUIRE(next == D, "the maps must fill the flat width");
  return GM_OK;
}

template <typename T, typename R>
int df_prepare(DfArgs<T, R>& a, const R* q, const R* k, const T* lambda, const T* records, const int64_t* desc,
               const int64_t* row_ptr, int64_t n_targets, int64_t n_sources, int64_t n_edges, int64_t D,
               int64_t orders, int64_t F, int64_t H, double scale) {
  GM_REQUIRE(n_targets >= 0 && n_sources >= 0 && n_edges >= 0, "sizes must be non-negative");
  GM_REQUIRE(n_targets < (int64_t(1) << 31) && n_sources < (int64_t(1) << 31) && n_edges < (int64_t(1) << 31),
             "the records index nodes and edges in 32 bits");
  const int rc = parse_maps(desc, F, H, D, orders, a.L);
  if (rc != GM_OK) return rc;
  if (n_targets > 0) GM_REQUIRE(q && row_ptr && lambda, "q, lambda and row_ptr must be device pointers");
  if (n_edges > 0) GM_REQUIRE(k && records, "k and the records must be device pointers");
  a.q = q;
  a.k = k;
  a.lambda = lambda;
  a.records = records;
  a.row_ptr = row_ptr;
  a.n_targets = n_targets;
  a.n_sources = n_sources;
  a.n_edges = n_edges;
  a.scale = (T)(scale * kLog2e);
  a.gradient_scale = (T)scale;
  return GM_OK;
}

// The rows' classes (order null: the simple kernels), which the lane kernels must serve.
template <typename T, typename R>
int df_rows(const DfArgs<T, R>& a, const int32_t* order, const int64_t* counts, int64_t n, DfRows& rows) {
  rows = DfRows{order, {0, 0, 0}};
  if (!order) return GM_OK;
  GM_REQUIRE((std::is_same<T, float>::value) && df_slots(a.L) > 0, "the lane kernels do not serve this layout");
  GM_REQUIRE(counts, "the classes' counts (a host array of three) are required");
  int64_t sum = 0;
  for (int c = 0; c < 3; ++c) {
    GM_REQUIRE(counts[c] >= 0, "a class has a negative count");
    rows.count[c] = counts[c];
    sum += counts[c];
  }
  GM_REQUIRE(sum == n, "the classes must hold every row once");
  GM_REQUIRE(aligned(a.q, 16) && aligned(a.k, 16) && aligned(a.dq, 16) && aligned(a.dk, 16) && aligned(a.records, 8) &&
                 aligned(a.records_s, 8) && aligned(a.stats, 8),
             "the lane kernels take rows at multiples of 16 bytes, records and statistics of 8");
  return GM_OK;
}

template <typename T, typename R>
int differential_forward(const R* q, const R* k, const T* lambda, const T* records, const int64_t* desc,
                         const int64_t* row_ptr, const int32_t* order, const int64_t* counts, int64_t n_targets,
                         int64_t n_sources, int64_t n_edges, int64_t D, int64_t orders, int64_t F, int64_t H,
                         double scale, T* alpha, T* stats, void* stream) {
  DfArgs<T, R> a{};
  const int rc = df_prepare(a, q, k, lambda, records, desc, row_ptr, n_targets, n_sources, n_edges, D, orders, F, H,
                            scale);
  if (rc != GM_OK) return rc;
  if (n_targets == 0) return GM_OK;
  if (n_edges > 0) GM_REQUIRE(alpha, "alpha must be a device pointer");
  a.alpha = alpha;
  a.stats = stats;
  DfRows rows;
  const int status = df_rows(a, order, counts, n_targets, rows);
  if (status != GM_OK) return status;
  if constexpr (std::is_same<T, float>::value) {
    if (order) return df_launch_units(DfPass::Forward, a, rows, (hipStream_t)stream);
  }
  hipLaunchKernelGGL((differential_forward_generic<T, R>), dim3((unsigned)blocks_for(n_targets)), dim3(256), 0,
                     (hipStream_t)stream, a);
  return check_launch("differential_forward");
}

template <typename T, typename R>
int differential_backward(const T* g, const R* q, const R* k, const T* lambda, const T* records, const T* records_s,
                          const int64_t* desc, const int64_t* row_ptr, const int64_t* src_ptr, const int32_t* order,
                          const int64_t* counts, const int32_t* order_s, const int64_t* counts_s, int64_t n_targets,
                          int64_t n_sources, int64_t n_edges, int64_t D, int64_t orders, int64_t F, int64_t H,
                          double scale, const T* stats, T* rows, T* ds, double* partial, R* dq, R* dk, T* dlambda,
                          void* stream) {
  DfArgs<T, R> a{};
  const int rc = df_prepare(a, q, k, lambda, records, desc, row_ptr, n_targets, n_sources, n_edges, D, orders, F, H,
                            scale);
  if (rc != GM_OK) return rc;
  GM_REQUIRE(partial && dlambda, "partial and dlambda must be device pointers");
  if (n_targets > 0) GM_REQUIRE(stats && rows && dq, "stats, rows and dq must be device pointers");
  if (n_sources > 0) GM_REQUIRE(src_ptr && dk, "src_ptr and dk must be device pointers");
  if (n_edges > 0) GM_REQUIRE(g && records_s, "g and the sources' records must be device pointers");
  GM_REQUIRE(!order == !order_s || n_targets == 0 || n_sources == 0, "both sides' rows are in classes, or neither's");
  const bool lanes = order || order_s;
  if (n_edges > 0 && !lanes) GM_REQUIRE(ds, "ds must be a device pointer without the rows' classes");
  a.g = g;
  a.records_s = records_s;
  a.src_ptr = src_ptr;
  a.stats = const_cast<T*>(stats);  // read only here
  a.rows = rows;
  a.ds = ds;
  a.dq = dq;
  a.dk = dk;
  const hipStream_t s = (hipStream_t)stream;
  DfRows targets, sources;
  int status = df_rows(a, order, counts, n_targets, targets);
  if (status == GM_OK) status = df_rows(a, order_s, counts_s, n_sources, sources);
  if (status != GM_OK) return status;
  if constexpr (std::is_same<T, float>::value) {
    if (lanes) {
      status = df_launch_units(DfPass::BackwardTarget, a, targets, s);
      if (status == GM_OK) status = df_launch_units(DfPass::BackwardSource, a, sources, s);
      if (status != GM_OK) return status;
    }
  }
  if (n_targets > 0 && !lanes) {
    const dim3 grid((unsigned)blocks_for(n_targets));
    hipLaunchKernelGGL((differential_backward_scores_generic<T, R>), grid, dim3(256), 0, s, a);
    hipLaunchKernelGGL((differential_backward_target_generic<T, R>), grid, dim3(256), 0, s, a);
  }
  if (n_sources > 0 && !lanes)
    hipLaunchKernelGGL((differential_backward_source_generic<T, R>), dim3((unsigned)blocks_for(n_sources)), dim3(256),
                       0, s, a);
  hipLaunchKernelGGL(differential_lambda_partial<T>, dim3(kLambdaBlocks), dim3(256), 0, s, (const T*)rows, n_targets,
                     (int)H, partial);
  hipLaunchKernelGGL(differential_lambda_sum<T>, dim3((unsigned)H), dim3(64), 0, s, (const double*)partial,
                     kLambdaBlocks, (int)H, dlambda);
  return check_launch("differential_backward");
}

}  // namespace
}  // namespace gm

extern "C" int64_t gm_differential_partials(int64_t heads) { return gm::kLambdaBlocks * heads; }

extern "C" int gm_differential_slots(const int64_t* desc, int64_t F, int64_t H, int64_t D, int64_t orders,
                                     int64_t* slots) {
  GM_REQUIRE(slots, "slots must be a host pointer");
  gm::DfLayout L{};
  const int rc = gm::parse_maps(desc, F, H, D, orders, L);
  if (rc != GM_OK) return rc;
  *slots = gm::df_slots(L);
  return GM_OK;
}

// T: the arithmetic's type, R the rows'.
#define GM_DIFFERENTIAL_ENTRY(SFX, T, R)                                                                              \
  extern "C" int gm_differential_forward_##SFX(                                                                       \
      const R* q, const R* k, const T* lambda, const T* records, const int64_t* desc, const int64_t* row_ptr,         \
      const int32_t* order, const int64_t* counts, int64_t n_targets, int64_t n_sources, int64_t n_edges, int64_t D,  \
      int64_t orders, int64_t F, int64_t H, double scale, T* alpha, T* stats, void* stream) {                           \
    return gm::differential_forward<T, R>(q, k, lambda, records, desc, row_ptr, order, counts, n_targets, n_sources,  \
                                          n_edges, D, orders, F, H, scale, alpha, stats, stream);                       \
  }                                                                                                                   \
  extern "C" int gm_differential_backward_##SFX(                                                                      \
      const T* g, const R* q, const R* k, const T* lambda, const T* records, const T* records_s, const int64_t* desc, \
      const int64_t* row_ptr, const int64_t* src_ptr, const int32_t* order, const int64_t* counts,                    \
      const int32_t* order_s, const int64_t* counts_s, int64_t n_targets, int64_t n_sources, int64_t n_edges,         \
      int64_t D, int64_t orders, int64_t F, int64_t H, double scale, const T* stats, T* rows, T* ds, double* partial,  \
      R* dq, R* dk, T* dlambda, void* stream) {                                                                       \
    return gm::differential_backward<T, R>(g, q, k, lambda, records, records_s, desc, row_ptr, src_ptr, order,        \
                                           counts, order_s, counts_s, n_targets, n_sources, n_edges, D, orders, F, H, \
                                           scale, stats, rows, ds, partial, dq, dk, dlambda, stream);                  \
  }

GM_DIFFERENTIAL_ENTRY(f32, float, float)
GM_DIFFERENTIAL_ENTRY(f64, double, double)
GM_DIFFERENTIAL_ENTRY(bf16, float, uint16_t)
