// What the kernels of the softmax with a learned relative bias share: the heads' layout, the arguments.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "edge_units.hpp"
#include "heads.hpp"

namespace gm {

constexpr int kRelMaxBuckets = 256;  // a float record's word holds a bucket above its source's 24 bits

struct RelLayout : HeadsLayout {
  int orders;
};

// The backward's lane kernels take two neighbouring rows (targets, or sources) at a time, a pair, over the entries of
// both: an entry is a node that either row has an edge with, and the edge of each, so that a node's row is loaded once
// for two edges.  Words of an entry: the node; the first row's edge (-1: it has none); one left free; the second's
// edge; (cos, sin) of both edges for the orders 1 ..  What stands for entries past a pair's last, words of 0 and -inf in
// turn, so reads as node 0 without edges.
constexpr int kRelPairHead = 4;

// Rows (pairs, or targets) by length: `order` lists them in three classes, a workgroup a row in the first two, a wave a
// row in the last; (count of each).
struct RelRows {
  const int32_t* order;
  int64_t count[3];
};

// T: the arithmetic's type; rows of T, or of bfloat16 (uint16_t) with T = float.
template <typename T, typename R>
struct RelArgs {
  RelLayout L;
  int buckets;
  const R* q;
  const R* k;
  const T* table;          // (buckets, H)
  const T* records;        // (n_edges, 2 orders): source and bucket, bias / log 2, (cos, sin) of orders 1 ..
  const T* records_s;      // (n_edges, 2 orders): target, edge, (cos, sin) of orders 1 ..; sorted by source
  const int64_t* row_ptr;  // over targets
  const int64_t* src_ptr;  // over sources
  const float* pairs;      // the backward's lane kernels': entries of pairs of targets, and their CSR over the pairs
  const int64_t* pair_ptr;
  const float* pairs_s;    // of pairs of sources
  const int64_t* pair_ptr_s;
  const T* g;              // (n_edges, H)
  T* alpha;                // (n_edges, H); read by the backward
  T* ds;                   // (n_edges, H): the backward's workspace
  T* partial;              // (gm_relative_partial_rows, buckets, H): sums of ds
  R* dq;
  R* dk;
  int64_t n_targets, n_sources, n_edges;
  T scale;           // of the scores, in units of log 2
  T gradient_scale;  // of the scores
  uint32_t by_heads;  // 2^16 / H and one: lane / H is the upper half of its product
};

// Scores, their biases and their maxima are in units of log 2.
constexpr double kRelLog2e = 1.4426950408889634074;

// A record's first word: the source below, the bucket above.
__device__ __forceinline__ int rel_source(const float* word) { return *reinterpret_cast<const int*>(word) & 0xFFFFFF; }
__device__ __forceinline__ int rel_bucket(const float* word) { return *reinterpret_cast<const uint32_t*>(word) >> 24; }
__device__ __forceinline__ int rel_source(const double* word) {
  return (int)(*reinterpret_cast<const int64_t*>(word) & 0xFFFFFFFF);
}
__device__ __forceinline__ int rel_bucket(const double* word) {
  return (int)(*reinterpret_cast<const int64_t*>(word) >> 32);
}
// A node or an edge in a word of its own.
__device__ __forceinline__ int rel_index(const float* word) { return *reinterpret_cast<const int*>(word); }
__device__ __forceinline__ int rel_index(const double* word) {
  return (int)*reinterpret_cast<const int64_t*>(word);
}

constexpr int kRelTableRows = 2048;  // rows of sums of ds by bucket that the backward adds

// The lane kernels (relative_units.hip).
enum class RelPass { Forward, BackwardTarget, BackwardSource };

// The edge slots of a wave (64 over the units rounded up to a power of two), or 0 where the lane kernels do not serve
// the layout.
int rel_slots(const RelLayout& L);

// A head's copies (of orders 0, 1, 2) filled up to a layout that the lane kernels serve, or false.
bool rel_padded(const RelLayout& L, int (&copies)[3]);

int rel_launch_units(RelPass pass, const RelArgs<float, float>& a, const RelRows& rows, hipStream_t stream);
int rel_launch_units(RelPass pass, const RelArgs<float, uint16_t>& a, const RelRows& rows, hipStream_t stream);

}  // namespace gm
