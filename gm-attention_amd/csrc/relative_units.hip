// The lane kernels of the softmax with a learned relative bias for float rows, and the layouts they serve.
#include "relative_units.hpp"

namespace gm {

// Every frequency's unit is loaded as one piece of 1, 2 or 4 numbers: the row's width and the frequency's offset are
// multiples of it (and the table's address one of 16 bytes, which the entry points check).
int rel_slots(const RelLayout& L) {
  int per_map = 0, base[3];
  const int shape = rel::rel_shape(L, per_map, base);
  if (shape < 0) return 0;
  const rel::RelShape& u = rel::kRelShapes[shape];
  const int width[3] = {u.a0, 2 * u.a1, 2 * u.a2};
  for (int f = 0; f < 3; ++f)
    if (width[f] > 0 && (base[f] % width[f] != 0 || L.D % width[f] != 0)) return 0;
  return kWave / lanes_for(L.H * per_map);
}

// A head's copies (c0, c1, c2) filled up with zeros to whole units: the fewest numbers, then the fewest lanes, of the
// layouts that the lane kernels serve with tables of as many orders; false where there is none.
bool rel_padded(const RelLayout& L, int (&copies)[3]) {
  int c[3] = {0, 0, 0};
  for (int f = 0; f < L.F; ++f) {
    if (L.n[f] > 2) return false;
    c[L.n[f]] = L.a[f];
  }
  int best = 0, best_per = 0;
  for (const rel::RelShape& u : rel::kRelShapes) {
    if (L.orders != (u.a2 > 0 ? 3 : (u.a1 > 0 ? 2 : 1))) continue;
    for (int per = 1; per * L.H <= kWave; per *= 2) {
      const int p[3] = {per * u.a0, per * u.a1, per * u.a2}, numbers = p[0] + 2 * p[1] + 2 * p[2];
      if (p[0] < c[0] || p[1] < c[1] || p[2] < c[2]) continue;
      if (best && (numbers > best || (numbers == best && per >= best_per))) continue;
      RelLayout to{};
      to.H = L.H;
      to.orders = L.orders;
      for (int n = 0; n < 3; ++n) {
        if (p[n] == 0) continue;
        to.n[to.F] = n;
        to.a[to.F] = p[n];
        to.off[to.F] = to.D;
        to.D += L.H * p[n] * (n == 0 ? 1 : 2);
        ++to.F;
      }
      if (to.D > GM_ATTN_MAX_D || rel_slots(to) == 0) continue;
      best = numbers;
      best_per = per;
      for (int n = 0; n < 3; ++n) copies[n] = p[n];
    }
  }
  return best > 0;
}

int rel_launch_units(RelPass pass, const RelArgs<float, float>& a, const RelRows& rows, hipStream_t stream) {
  return rel::rel_launch_any<float>(pass, a, rows, stream);
}

}  // namespace gm
