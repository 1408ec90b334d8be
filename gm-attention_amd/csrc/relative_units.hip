#include "relative.hpp"

namespace gm {

int rel_slots(const RelLayout&) { return 0; }

int rel_launch_units(RelPass, const RelArgs<float, float>&, const RelRows&, hipStream_t) {
  return fail(GM_ERR_UNSUPPORTED, "relative: the lane kernels do not serve this layout");
}
int rel_launch_units(RelPass, const RelArgs<float, uint16_t>&, const RelRows&, hipStream_t) {
  return fail(GM_ERR_UNSUPPORTED, "relative: the lane kernels do not serve this layout");
}

}  // namespace gm
