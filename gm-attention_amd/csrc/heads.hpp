// The layout of rows of heads, as entry points read it from a descriptor.
#pragma once
#include <cstdint>

#include "common.hpp"

namespace gm {

constexpr int kHeadsMaxFreq = GM_ATTN_MAX_F;

// H heads side by side within each frequency: frequency f's order n, copies a a head, flat offset.
struct HeadsLayout {
  int F, H, D;
  int n[kHeadsMaxFreq], a[kHeadsMaxFreq], off[kHeadsMaxFreq];
};

// desc: a host pointer to (F, 5) int64, of each frequency its order, the copies a head, the flat offset, -, and 1 at
// frequency 0, 2 above; the orders rise and the frequencies fill the D columns one after the other.
inline int parse_heads(const int64_t* desc, int64_t F, int64_t H, int64_t max_heads, int64_t D, HeadsLayout& L) {
  GM_REQUIRE(desc != nullptr, "desc must be a host pointer to (F, 5) int64");
  GM_REQUIRE(F >= 1 && F <= kHeadsMaxFreq, "desc must have 1 to 8 frequency rows");
  GM_REQUIRE(H >= 1 && H <= max_heads, "at most " + std::to_string(max_heads) + " heads");
  GM_REQUIRE(D >= 1 && D <= GM_ATTN_MAX_D, "D must be in [1, 1024]");
  L.F = (int)F;
  L.H = (int)H;
  L.D = (int)D;
  int64_t next = 0;
  for (int f = 0; f < F; ++f) {
    const int64_t* row = desc + f * GM_ATTN_DESC;
    GM_REQUIRE(row[0] >= 0 && row[0] < (int64_t(1) << 31), "a descriptor frequency is out of range");
    GM_REQUIRE(f == 0 || row[0] > desc[(f - 1) * GM_ATTN_DESC], "the descriptor's frequencies must rise");
    GM_REQUIRE(row[4] == (row[0] == 0 ? 1 : 2), "descriptor dim must be 1 at frequency 0 and 2 above");
    GM_REQUIRE(row[1] >= 1 && row[1] <= GM_ATTN_MAX_D && row[2] == next,
               "the descriptor's rows must hold copies and follow each other");
    next += H * row[1] * row[4];
    GM_REQUIRE(next <= D, "a descriptor row runs past the flat width D");
    L.n[f] = (int)row[0];
    L.a[f] = (int)row[1];
    L.off[f] = (int)row[2];
  }
  GM_REQUIRE(next == D, "the heads must fill the flat width");
  return GM_OK;
}

}  // namespace gm
