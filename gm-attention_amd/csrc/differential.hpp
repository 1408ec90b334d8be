// What the differential softmax's kernels share: the maps' layout, the arguments.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace gm {

constexpr int kDfMaxFreq = GM_ATTN_MAX_F;

// The 2 H maps in the rows: frequency f's order n, copies a a map, flat offset.
struct DfLayout {
  int F, H, P, D, orders;
  int n[kDfMaxFreq], a[kDfMaxFreq], off[kDfMaxFreq];
};

// The rows (targets, or sources) as the lane kernels take them: `order` lists them in three classes, those of 16 waves
// each, of four, of one; (count of each).
struct DfRows {
  const int32_t* order;
  int64_t count[3];
};

// T: the arithmetic's type; rows of T, or of bfloat16 (uint16_t) with T = float.
template <typename T, typename R>
struct DfArgs {
  DfLayout L;
  const R* q;
  const R* k;
  const T* lambda;         // (H)
  const T* records;        // (n_edges, 2 orders): other node, bias / log 2, (cos, sin) of orders 1 ..
  const T* records_s;      // (n_edges, 2 + 2 orders): target, edge, bias, 0, (cos, sin) of orders 1 ..
  const int64_t* row_ptr;  // over targets
  const int64_t* src_ptr;  // over sources
  const T* g;              // (n_edges, H)
  T* alpha;                // (n_edges, H)
  T* stats;                // (n_targets, 2 H, 2): m, the largest s, and 1 / sum 2^(s - m) (zeros where no edge is inside)
  T* rows;                 // (n_targets, 2 H, 3): both beside T, the backward's workspace
  T* ds;                   // (n_edges, 2 H): the generic backward's workspace
  R* dq;
  R* dk;
  int64_t n_targets, n_sources, n_edges;
  T scale;           // of the scores, in units of log 2
  T gradient_scale;  // of the scores
};

// Scores, their biases and their maxima are in units of log 2: a weight is 2^(s - m) / sum 2^(s - m), in the backward
// as in the forward.  (m + log2 of the sum as one number is as wrong as that number's spacing: beside a bias of -1e9 by
// more than the sum itself, and the backward's weights were not the forward's.)
constexpr double kLog2e = 1.4426950408889634074;

__device__ __forceinline__ float df_exp2(float x) { return exp2f(x); }
__device__ __forceinline__ double df_exp2(double x) { return exp2(x); }
__device__ __forceinline__ float df_widen(float x) { return x; }
__device__ __forceinline__ double df_widen(double x) { return x; }
__device__ __forceinline__ float df_widen(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }
__device__ __forceinline__ void df_narrow(float v, float& o) { o = v; }
__device__ __forceinline__ void df_narrow(double v, double& o) { o = v; }
__device__ __forceinline__ void df_narrow(float v, uint16_t& o) {  // to nearest even
  o = __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
}

// The lane kernels (differential_units.hip): a map's copies as `per_map` units of (A0, A1, A2) copies, one lane a unit.
enum class DfPass { Forward, BackwardTarget, BackwardSource };

// The edge slots of a wave (64 over the units rounded up to a power of two), or 0 where the lane kernels do not serve
// the layout.
int df_slots(const DfLayout& L);

int df_launch_units(DfPass pass, const DfArgs<float, float>& a, const DfRows& rows, hipStream_t stream);
int df_launch_units(DfPass pass, const DfArgs<float, uint16_t>& a, const DfRows& rows, hipStream_t stream);

}  // namespace gm
