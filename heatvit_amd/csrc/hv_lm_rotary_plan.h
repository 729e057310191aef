// hv_lm_rotary_plan.h -- how many lanes a head of the rotary kernels takes. Code without HIP,
// so that tests can run it on the host.
#pragma once

#include "hv_lm_paged.h"

namespace hv {

// Lanes that hold eight pairs each, and those that hold sixteen elements of what follows them:
// 65 at most in all, for heads of up to 1024 elements whose two parts both end within a lane.
HV_HD int rotary_pair_lanes(int pairs) { return (pairs + 7) / 8; }
HV_HD int rotary_lanes(int pairs, int width) {
  return rotary_pair_lanes(pairs) + (width - 2 * pairs + 15) / 16;
}

}  // namespace hv
