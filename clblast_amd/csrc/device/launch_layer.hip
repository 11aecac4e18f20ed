// =================================================================================================
// Device-layer entry points of the layer products: validation of the descriptor, plan, dispatch by storage type.
// =================================================================================================
#include "device/launch_layer.hpp"

namespace {

using clbh::PlanLayer;

int Units() {
  int units = 0;
  return (clbh_compute_units(&units) == 0 && units > 0) ? units : 256;
}

// What a plan can be made for: a known type, sizes and numbers of groups within the limits
bool ValidSizes(const clbh_layer_desc& d) {
  if (d.type != CLBH_TYPE_FP16 && d.type != CLBH_TYPE_BF16 && d.type != CLBH_TYPE_FP32) { return false; }
  if (d.m <= 0 || d.n <= 0 || (d.k <= 0 && d.upstream == nullptr)) { return false; }
  if (d.m > CLBH_LAYER_MAX_SIZE || d.n > CLBH_LAYER_MAX_SIZE || d.k > CLBH_LAYER_MAX_SIZE) { return false; }
  if (!clbh::LayerOperandsReachable(d)) { return false; }
  if (d.grouping == CLBH_GROUPS_NONE) { return true; }
  if (d.grouping != CLBH_GROUPS_BY_ROWS && d.grouping != CLBH_GROUPS_BY_DEPTH) { return false; }
  if (d.groups <= 0 || d.groups > CLBH_LAYER_MAX_GROUPS) { return false; }
  return (d.grouping == CLBH_GROUPS_BY_ROWS ? d.n : d.k) < CLBH_LAYER_MAX_GROUPED;
}

// Every access of the kernels follows from these: sizes, leading dimensions that hold a line, pointers where they are used
bool ValidLayer(const clbh_layer_desc& d) {
  const auto aligned = [&](const void* pointer) {
    return reinterpret_cast<unsigned long long>(pointer) % (d.type == CLBH_TYPE_FP32 ? 4 : 2) == 0;
  };
  if (!ValidSizes(d) || d.activation < 161 || d.activation > 165) { return false; }
  if (d.grouping != CLBH_GROUPS_NONE && (d.offsets == nullptr || reinterpret_cast<unsigned long long>(d.offsets) % 8 != 0)) { return false; }
  if (!aligned(d.c) || !aligned(d.pre) || !aligned(d.residual) || !aligned(d.bias) || !aligned(d.upstream) || !aligned(d.bias_gradient) || !aligned(d.a) || !aligned(d.b)) { return false; }
  if (d.c != nullptr && d.c_ld < d.m) { return false; }
  if (d.pre != nullptr && d.pre_ld < d.m) { return false; }
  if (!d.gradient && d.beta != 0.0f && (d.residual == nullptr || d.residual_ld < d.m)) { return false; }
  if (d.gradient && (d.bias != nullptr || d.beta != 0.0f || (d.pre == nullptr && d.activation != 161))) { return false; }
  if (!d.gradient && d.bias_gradient != nullptr) { return false; }
  if (d.upstream != nullptr) {
    return d.gradient && d.grouping != CLBH_GROUPS_BY_DEPTH && d.upstream_ld >= d.m && (d.c != nullptr || d.bias_gradient != nullptr);
  }
  if (d.a == nullptr || d.b == nullptr || d.c == nullptr) { return false; }
  const bool by_rows = d.grouping == CLBH_GROUPS_BY_ROWS, by_depth = d.grouping == CLBH_GROUPS_BY_DEPTH;
  if (d.a_ld < (d.a_kcontig ? d.k : d.m) || d.b_ld < (d.b_kcontig ? d.k : d.n)) { return false; }
  if (by_rows && (!d.b_kcontig || d.a_stride < 0 || d.bias_stride < 0 || d.gradient)) { return false; }
  if (by_depth && (d.a_kcontig || d.b_kcontig || d.c_stride < 0 || d.gradient || d.bias != nullptr || d.pre != nullptr || d.activation != 161)) { return false; }
  return !by_depth || d.beta == 0.0f || d.residual == d.c;
}

}  // namespace

extern "C" {

size_t clbh_layer_workspace_bytes(const clbh_layer_desc* desc) {
  return (desc != nullptr && ValidSizes(*desc)) ? PlanLayer(*desc, Units()).workspace_bytes : 0;
}

int clbh_layer_launch(const clbh_layer_desc* desc, hipStream_t stream) {
  if (desc == nullptr || !ValidLayer(*desc)) { return hipErrorInvalidValue; }
  const auto plan = PlanLayer(*desc, Units());
  if (plan.workspace_bytes > 0 && (desc->workspace == nullptr || desc->workspace_bytes < plan.workspace_bytes)) { return hipErrorInvalidValue; }
  switch (desc->type) {
    case CLBH_TYPE_FP16: return clbh::LaunchLayerF16(*desc, plan, stream);
    case CLBH_TYPE_BF16: return clbh::LaunchLayerBF16(*desc, plan, stream);
    default: return clbh::LaunchLayerF32(*desc, plan, stream);
  }
}

}  // extern "C"
