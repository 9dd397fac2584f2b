// Dense-layer kernels (linear_tile.h) for one element type.
#include "linear_tile.h"

namespace dtf {
const LinLaunch& lin_launch_f32() {
  static const LinLaunch l = lin_make_launch<MM_F32>();
  return l;
}
}  // namespace dtf
