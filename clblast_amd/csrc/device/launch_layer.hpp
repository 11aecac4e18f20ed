// =================================================================================================
// Instances and launches of the layer products for one storage type (see clbh_layer_desc).
// =================================================================================================
#ifndef CLBLAST_HIP_DEVICE_LAUNCH_LAYER_HPP_
#define CLBLAST_HIP_DEVICE_LAUNCH_LAYER_HPP_

#include <hip/hip_runtime.h>

#include <climits>

#include "clbh_device.h"
#include "device/layer_plans.hpp"
#include "kernels/layer_gemm.hpp"
#include "kernels/layer_rows.hpp"

namespace clbh {

int LaunchLayerF16(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream);
int LaunchLayerBF16(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream);
int LaunchLayerF32(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream);

inline LayerArgs MakeLayerArgs(const clbh_layer_desc& d, const LayerPlan& plan) {
  LayerArgs p{};
  p.a = d.a;
  p.b = d.b;
  p.c = d.c;
  p.a_ld = d.a_ld;
  p.b_ld = d.b_ld;
  p.c_ld = d.c_ld;
  p.a_stride = d.a_stride;
  p.c_stride = d.c_stride;
  p.m = d.m;
  p.n = d.n;
  p.k = d.k;
  p.alpha = d.alpha;
  p.beta = d.beta;
  p.bias = d.bias;
  p.bias_stride = d.bias_stride;
  p.pre = d.pre;
  p.pre_ld = d.pre_ld;
  p.residual = d.residual;
  p.residual_ld = d.residual_ld;
  p.activation = d.activation;
  p.gradient = d.gradient;
  p.grouping = d.grouping;
  p.groups = d.groups;
  p.offsets = d.offsets;
  const long long size = (d.type == CLBH_TYPE_FP32) ? 4 : 2;
  const auto movable = [&](const void* pointer, const long long ld) {
    return pointer == nullptr || (reinterpret_cast<unsigned long long>(pointer) % 4 == 0 && (ld * size) % 4 == 0);
  };
  p.vector_rows = movable(d.c, d.c_ld) && movable(d.c, d.c_stride) && movable(d.pre, d.pre_ld) &&
                  (d.beta == 0.0f || movable(d.residual, d.residual_ld)) && movable(d.upstream, d.upstream_ld);
  if (plan.splits > 1) {
    p.split_chunk = plan.chunk;
    p.partials = static_cast<float*>(d.workspace);
  }
  if (d.bias_gradient != nullptr) {
    p.bias_partials = reinterpret_cast<float*>(static_cast<char*>(d.workspace) + plan.partial_bytes);
  }
  return p;
}

template <typename Config, bool A_KC, bool B_KC>
int LaunchLayerTile(const clbh_layer_desc& d, const LayerPlan& plan, const LayerArgs& args, hipStream_t stream) {
  if (Config::TILE_M != plan.tile.tile_m || Config::TILE_N != plan.tile.tile_n) { return hipErrorInvalidValue; }
  const long long blocks = plan.tiles_m * plan.tiles_n * ((d.grouping == CLBH_GROUPS_BY_DEPTH) ? d.groups : 1);
  if (blocks > INT_MAX) { return hipErrorInvalidConfiguration; }
  auto kernel = LayerGemmKernel<Config, A_KC, B_KC>;
  constexpr int lds_bytes = Config::LDS_BYTES;
  if (lds_bytes > 48 * 1024) {
    static const hipError_t attribute_status =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds_bytes);
    if (attribute_status != hipSuccess) { return static_cast<int>(attribute_status); }
  }
  kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(plan.splits)), dim3(Config::THREADS), lds_bytes, stream>>>(
      args, static_cast<int>(plan.tiles_m), static_cast<int>(plan.tiles_n));
  return static_cast<int>(hipGetLastError());
}

template <typename Config>
int LaunchLayerConfig(const clbh_layer_desc& d, const LayerPlan& plan, const LayerArgs& args, hipStream_t stream) {
  switch ((d.a_kcontig ? 2 : 0) | (d.b_kcontig ? 1 : 0)) {
    case 0: return LaunchLayerTile<Config, false, false>(d, plan, args, stream);
    case 1: return LaunchLayerTile<Config, false, true>(d, plan, args, stream);
    case 2: return LaunchLayerTile<Config, true, false>(d, plan, args, stream);
    default: return LaunchLayerTile<Config, true, true>(d, plan, args, stream);
  }
}

template <typename T>
int LaunchLayerProduct(const clbh_layer_desc& d, const LayerPlan& plan, const LayerArgs& args, hipStream_t stream) {
  switch (plan.tile.variant) {
    case 1:
      if constexpr (sizeof(T) == 2) { return LaunchLayerConfig<LayerConfig<T, 2, 4, 4, 2, 2>>(d, plan, args, stream); }
      else { return hipErrorInvalidValue; }
    case 2: return LaunchLayerConfig<LayerConfig<T, 2, 2, 4, 2, 2>>(d, plan, args, stream);
    case 3: return LaunchLayerConfig<LayerConfig<T, 2, 2, 1, 1, 4>>(d, plan, args, stream);
    case 4: return LaunchLayerConfig<LayerConfig<T, 4, 1, 1, 1, 4>>(d, plan, args, stream);
    default: return LaunchLayerConfig<LayerConfig<T, 2, 2, 2, 2, 2>>(d, plan, args, stream);
  }
}

template <typename T, int V>
int LaunchLayerRowsOf(const clbh_layer_desc& d, const LayerPlan& plan, const LayerArgs& args, hipStream_t stream) {
  LayerRowsArgs q{};
  q.layer = args;
  q.upstream = d.upstream;
  q.upstream_ld = d.upstream_ld;
  q.ranges = (d.upstream != nullptr) ? 1 : plan.splits;
  q.chunk = plan.rows_chunk;
  const long long column_blocks = (static_cast<long long>(d.m) + 64 * V - 1) / (64 * V);
  if (column_blocks * plan.rows_chunks > INT_MAX) { return hipErrorInvalidConfiguration; }
  q.column_blocks = static_cast<int>(column_blocks);
  LayerRowsKernel<T, V><<<dim3(static_cast<unsigned>(column_blocks * plan.rows_chunks)), dim3(kLayerRowsThreads), 0, stream>>>(q);
  return static_cast<int>(hipGetLastError());
}

template <typename T>
int LaunchLayerTyped(const clbh_layer_desc& d, const LayerPlan& plan, hipStream_t stream) {
  const auto args = MakeLayerArgs(d, plan);
  const bool elementwise = d.upstream != nullptr || plan.splits > 1;
  if (d.upstream == nullptr) {
    const int status = LaunchLayerProduct<T>(d, plan, args, stream);
    if (status != 0) { return status; }
  }
  if (elementwise) {
    constexpr int V = 16 / sizeof(T);
    const int status = args.vector_rows ? LaunchLayerRowsOf<T, V>(d, plan, args, stream) : LaunchLayerRowsOf<T, 1>(d, plan, args, stream);
    if (status != 0) { return status; }
  }
  if (d.bias_gradient != nullptr) {
    const long long rows_of_sums = elementwise ? plan.rows_chunks : plan.tiles_n;
    const bool grouped = d.grouping == CLBH_GROUPS_BY_ROWS;
    const int groups = grouped ? d.groups : 1;
    const dim3 grid(static_cast<unsigned>((static_cast<long long>(d.m) + 63) / 64), static_cast<unsigned>(groups < 65535 ? groups : 65535));
    LayerColumnSumsKernel<T><<<grid, dim3(kLayerRowsThreads), 0, stream>>>(
        args.bias_partials, static_cast<int>(rows_of_sums), d.m, grouped ? d.offsets : nullptr, groups, d.n,
        elementwise ? plan.rows_chunk : plan.tile.tile_n, static_cast<T*>(d.bias_gradient), static_cast<long long>(d.m));
    return static_cast<int>(hipGetLastError());
  }
  return 0;
}

}  // namespace clbh

#endif  // CLBLAST_HIP_DEVICE_LAUNCH_LAYER_HPP_
