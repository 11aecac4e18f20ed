// =================================================================================================
// bf16 instances of the layer products.
// =================================================================================================
#include "device/launch_layer.hpp"

namespace clbh {
int LaunchLayerBF16(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream) { return LaunchLayerTyped<__bf16>(d, plan, stream); }
}  // namespace clbh
