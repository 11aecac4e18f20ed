// =================================================================================================
// fp16 instances of the layer products.
// =================================================================================================
#include "device/launch_layer.hpp"

namespace clbh {
int LaunchLayerF16(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream) { return LaunchLayerTyped<_Float16>(d, plan, stream); }
}  // namespace clbh
