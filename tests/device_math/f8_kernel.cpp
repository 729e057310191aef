// The rule that picks a product's kernel, for the tests.
#include "hv_lm_plan.h"

extern "C" int f8_kernel(int f32, int m, int n, long long lda) {
  return (int)hv::f8_kernel(f32 != 0, m, n, lda);
}
