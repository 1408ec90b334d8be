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

int rel_launch_units(RelPass pass, const RelArgs<float, float>& a, const RelRows& rows, hipStream_t stream) {
  return rel::rel_launch_any<float>(pass, a, rows, stream);
}

}  // namespace gm
