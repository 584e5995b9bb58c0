// The block-scaled attention's instances for f32 queries.
#include "scaled_attention.h"

namespace vpa {

hipError_t launch_scaled_attention_f32(const ScaledArgs& a, const CacheGeom& g, const ScaledPlan& p,
                                      hipStream_t stream) {
  return launch_scaled<float>(a, g, p, stream);
}

}  // namespace vpa
