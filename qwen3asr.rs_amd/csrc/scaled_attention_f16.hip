// The block-scaled attention's instances for f16 queries.
#include "scaled_attention.h"

namespace vpa {

hipError_t launch_scaled_attention_f16(const ScaledArgs& a, const CacheGeom& g, const ScaledPlan& p,
                                      hipStream_t stream) {
  return launch_scaled<f16_t>(a, g, p, stream);
}

}  // namespace vpa
