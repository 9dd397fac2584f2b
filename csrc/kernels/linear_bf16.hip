// Dense-layer kernels (linear_tile.h) for one element type.
#include "linear_tile.h"

namespace dtf {
const LinLaunch& lin_launch_bf16() {
  static const LinLaunch l = lin_make_launch<MM_BF16>();
  return l;
}
}  // namespace dtf
