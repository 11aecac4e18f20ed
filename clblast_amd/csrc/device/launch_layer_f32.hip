// =================================================================================================
// fp32 instances of the layer products.
// =================================================================================================
#include "device/launch_layer.hpp"

namespace clbh {
int LaunchLayerF32(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream) { return LaunchLayerTyped<float>(d, plan, stream); }
}  // namespace clbh
