// hv_lm_attn_f16.hip -- the attention kernels of float16 heads.
#include "hv_lm_attn_tile.h"

int hv::attend_f16(const LmAttnArgs &a, bool paged, bool q8, void *workspace, size_t bytes,
                    hipStream_t s) {
  return attend_any<f16>(a, paged, q8, workspace, bytes, s);
}
