// The lane kernels of the softmax with a learned relative bias for bfloat16 rows.
#include "relative_units.hpp"

namespace gm {

int rel_launch_units(RelPass pass, const RelArgs<float, uint16_t>& a, const RelRows& rows, hipStream_t stream) {
  return rel::rel_launch_any<uint16_t>(pass, a, rows, stream);
}

}  // namespace gm
